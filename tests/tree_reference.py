"""Plain float64 form of the tree attention, token by token, for the tests."""
import math

import torch


def depths(parents):
    """Depth of every token of one sequence, -1 where there is none."""
    out = []
    for i, p in enumerate(parents):
        out.append(0 if p == -1 else out[p] + 1 if 0 <= p < i and out[p] >= 0 else -1)
    return out


def turn(x, cos, sin, rows, axis, interleaved):
    """x (heads, d) in fp32 steps, rounded once: pair i by table row rows[axis[i]]."""
    y = x.float().clone()
    pairs = cos.shape[1]
    i = torch.arange(pairs)
    r = torch.tensor([min(max(rows[a], 0), cos.shape[0] - 1) for a in axis])
    c, s = cos.float()[r, i], sin.float()[r, i]
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    a, b = x.float()[:, lo], x.float()[:, hi]
    y[:, lo], y[:, hi] = a * c - b * s, a * s + b * c
    return y.to(x.dtype)


def tree_attention(q, kc, vc, k, v, parents, lens, table=None, batch_idx=None, cos=None, sin=None, positions=None, axis=None,
                   interleaved=True, scale=None, left=-1, softcap=0.0):
    """CPU tensors; kc, vc are changed in place.  -> out, lse, A (float64), A = sum of p |v|, which scales the error of P."""
    B, T, Hq, D = q.shape
    Hkv = kc.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    page = kc.shape[1]
    cap = page * table.shape[1] if table is not None else page
    out, mag = torch.zeros(B, T, Hq, D, dtype=torch.float64), torch.zeros(B, T, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), math.inf, dtype=torch.float64)

    def place(b, row):
        if row >= cap:
            return None
        if table is None:
            return (int(batch_idx[b]) if batch_idx is not None else b), row
        pg = int(table[b, row // page])
        return (pg, row % page) if 0 <= pg < kc.shape[0] else None

    todo = []
    for b in range(B):
        L = max(0, min(int(lens[b]), cap))
        ds = depths([int(x) for x in parents[b]])
        qb = q[b].clone()
        for t in range(T):
            rows = None
            if cos is not None:
                rows = [L + max(ds[t], 0)] * 4 if positions is None else [int(positions[a, b, t]) for a in range(positions.shape[0])]
                ax = axis if axis is not None else [0] * cos.shape[1]
                qb[t] = turn(q[b, t], cos, sin, rows, ax, interleaved)
            at = place(b, L + t)
            if ds[t] >= 0 and at is not None and k is not None:
                kc[at] = turn(k[b, t], cos, sin, rows, ax, interleaved) if cos is not None else k[b, t]
                vc[at] = v[b, t]
        todo.append((b, L, ds, qb))
    for b, L, ds, qb in todo:
        prefix = [place(b, j) for j in range(L)]
        kp = torch.stack([kc[p].double() if p else torch.zeros(Hkv, D, dtype=torch.float64) for p in prefix]) if L else torch.zeros(0, Hkv, D, dtype=torch.float64)
        vp = torch.stack([vc[p].double() if p else torch.zeros(Hkv, D, dtype=torch.float64) for p in prefix]) if L else torch.zeros(0, Hkv, D, dtype=torch.float64)
        for t in range(T):
            if ds[t] < 0:
                continue
            lo = 0 if left < 0 else min(L, max(0, L + ds[t] - left))
            mine, cur, steps = [], t, 0
            while cur >= 0 and (left < 0 or steps <= left):
                if place(b, L + cur) is not None:
                    mine.append(place(b, L + cur))
                cur, steps = int(parents[b][cur]), steps + 1
            kk = torch.cat([kp[lo:]] + [kc[p].double()[None] for p in mine])
            vv = torch.cat([vp[lo:]] + [vc[p].double()[None] for p in mine])
            if not len(kk):
                continue
            s = torch.einsum("hgd,nhd->hgn", qb[t].double().reshape(Hkv, G, D), kk).reshape(Hq, -1) * scale
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            lse[b, :, t] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[b, :, t, None]).reshape(Hkv, G, -1)
            out[b, t] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(Hq, D)
            mag[b, t] = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(Hq, D)
    return out, lse, mag


def out_bound(out, mag, dtype):
    """Elementwise bound of the kernels' error.  Roundings to the input type, eps / 2 each: the output itself, and P before
    the second product (at most eps / 2 of sum p |v|).  2^-12 of sum p |v| is for all that is done in fp32: scores of up to 256
    products, the exponential's approximation, the row sum and the joining of splits, each below 2^-15."""
    half = torch.finfo(dtype).eps / 2
    return half * out.abs() + (half + 2.0 ** -12) * 1.01 * mag + 1e-6
