"""The operators around the attention layers in 64 bits, and how far a kernel of 32-bit sums may be off.  Test infrastructure.

`bound` arrays are worst cases by arithmetic, element by element.  u is what one rounding of a formed value (a probability,
a share, a score's gradient, an output) is off by at most, relative to the value: 2^-8 for bf16.  For fp32 kernels u stands
for all the roundings of a sum of n terms, n 2^-24.  Scores are fp32 sums of D products: off by at most
(D + 8) 2^-24 sum |q k| each, which every probability carries as a relative error (`slack`).

A capped score is off by at most 4e-7 min(cap, |s|) next to bf16, s the score in front of the cap: below the cap tanh is x + x^3 P(x^2),
whose fit (8e-8), argument (two roundings), polynomial (0.33 2^-23) and last rounding come to 3e-7 of x; past it 1 - 2 / (1 + e^2x), whose
exponential (2^-22, times 0.12 at x = -1), reciprocal (2^-23) and sums come to 3.7e-7 of the cap.  Up to caps of 1024 a score below the
cap may take the second form, off by that much of the cap (`cap_error`): a tenth of a probability's rounding."""

from __future__ import annotations

import math

import torch

EPS = 1e-9


def visible(seq, documents=None, prefix=None, device="cpu"):
    """(seq, seq) truth values of one sequence: the row's query sees the column's key."""
    i = torch.arange(seq, device=device)
    see = i[:, None] >= i[None, :]
    if prefix is not None:
        see = see | (i[None, :] < prefix)
    if documents is not None:
        see = see & (documents[:, None] == documents[None, :]) & (documents >= 0)[:, None]
    return see


def _unit(dtype, terms):
    return 2.0 ** -8 if dtype == torch.bfloat16 else (terms + 64) * 2.0 ** -24


def cap_error(s, softcap):
    return 4e-7 * (softcap if softcap <= 1024 else s.abs().clamp(max=softcap))


def attention(q, k, v, dout=None, softcap=None, slopes=None, documents=None, prefix=None):
    """((out, dq, dk, dv), bounds) of masked softmax attention, or (out,) and its bound without dout."""
    dtype, (batch, heads, seq, dim) = q.dtype, q.shape
    group = heads // k.shape[1]
    u = _unit(dtype, seq + dim)
    scale = dim ** -0.5
    q64, k64, v64 = (x.detach().double() for x in (q, k, v))
    shapes = (q64, q64, k64, v64) if dout is not None else (q64,)
    got, off = [torch.zeros_like(x) for x in shapes], [torch.zeros_like(x) for x in shapes]
    far = (torch.arange(seq, device=q.device)[:, None] - torch.arange(seq, device=q.device)[None, :]).abs().double()
    for b in range(batch):
        see = visible(seq, None if documents is None else documents[b], None if prefix is None else prefix[b], q.device)
        for h in range(heads):
            g = h // group
            # (rows that no one sees may hold anything)
            qs, ks, vs = (torch.where(torch.isfinite(x), x, 0.0) for x in (q64[b, h], k64[b, g], v64[b, g]))
            c = qs @ ks.T * scale
            size = qs.abs() @ ks.abs().T * scale
            t, capped = torch.zeros_like(c), 0.0
            if softcap is not None:
                capped = cap_error(c, softcap)
                t = torch.tanh(c / softcap)
                c = softcap * t
            a = c if slopes is None else c - slopes[h].double() * far
            a = a.masked_fill(~see, -math.inf)
            top = a.amax(-1, keepdim=True)
            e = torch.exp(a - torch.where(torch.isfinite(top), top, 0.0))
            mass = e.sum(-1, keepdim=True)
            p = e / torch.where(mass > 0, mass, 1.0)
            # a score's error, also through the cap and the distance's product
            wrong = (dim + 8) * 2.0 ** -24 * size + capped + 2.0 ** -22 * torch.where(see, a.abs(), 0.0)
            slack = 2 * wrong.masked_fill(~see, 0.0).amax(-1, keepdim=True) + 2.0 ** -20
            out = p @ vs
            spread = p @ vs.abs()
            # weights off by e_j each, divided by their own sum, leave sum p_j e_j (v_j - out), at most u (spread + |out|); out's rounding is u |out|
            far_out = (u + slack) * spread + 2 * u * out.abs()
            got[0][b, h], off[0][b, h] = out, far_out
            if dout is None:
                continue
            do = torch.where(torch.isfinite(dout[b, h].double()), dout[b, h].double(), 0.0)
            do = do * see.any(-1, keepdim=True)
            dp = do @ vs.T
            delta = (do * out).sum(-1, keepdim=True)
            delta_off = (do.abs() * far_out).sum(-1, keepdim=True) + (dim + 8) * 2.0 ** -24 * (do.abs() * spread).sum(-1, keepdim=True)
            ds = p * (dp - delta) * (1 - t * t)
            ds_off = p * (delta_off + (dim + 8) * 2.0 ** -24 * (do.abs() @ vs.abs().T)) + (u + slack) * ds.abs() \
                + p * (dp - delta).abs() * 4e-6
            dq, dk, dv = scale * ds @ ks, scale * ds.T @ qs, p.T @ do
            got[1][b, h], off[1][b, h] = dq, scale * ds_off @ ks.abs() + u * dq.abs()
            got[2][b, g] += dk
            off[2][b, g] += scale * ds_off.T @ qs.abs()
            got[3][b, g] += dv
            off[3][b, g] += ((u + slack) * p).T @ do.abs()
    if dout is not None:
        for x in (2, 3):
            off[x] += u * got[x].abs()
    return tuple(got), tuple(off)


def tree_nodes(q, k, v, cache_k, cache_v, length, parents, softcap=None, slopes=None, committed=None):
    """Node by node, each after its parent: (out, bound, bids, their bound); bids (B, H, N, length + N) double.
    With committed (B, H, capacity): the dilution operator."""
    batch, heads, nodes, dim = q.shape
    group = heads // k.shape[1]
    u = _unit(q.dtype, length + nodes + dim)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    bids = torch.zeros(batch, heads, nodes, length + nodes, dtype=torch.float64, device=q.device)
    bids_off = torch.zeros_like(bids)
    for b in range(batch):
        tree = parents if not isinstance(parents[0], (list, tuple)) else parents[b]
        for h in range(heads):
            g = h // group
            keys = torch.cat((cache_k[b, g, :length], k[b, g])).double()
            vals = torch.cat((cache_v[b, g, :length], v[b, g])).double()
            branches, demands, demand_offs = [], [], []
            for x in range(nodes):
                up = tree[x] if 0 <= tree[x] < x else -1
                branch = (branches[up] if up >= 0 else []) + [x]
                branches.append(branch)
                seen = list(range(length)) + [length + y for y in branch]
                at = torch.tensor(seen, device=q.device)
                s = keys[at] @ q[b, h, x].double() * dim ** -0.5
                size = keys[at].abs() @ q[b, h, x].double().abs() * dim ** -0.5
                capped = 0.0
                if softcap is not None:
                    capped = cap_error(s, softcap)
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - slopes[h].double() * torch.arange(len(seen) - 1, -1, -1, device=q.device)
                p = torch.softmax(s, 0)
                slack = 2 * ((dim + 8) * 2.0 ** -24 * size + capped + 2.0 ** -22 * s.abs()).amax() + 2.0 ** -20
                bids[b, h, x, at] = p
                bids_off[b, h, x, at] = slack * p
                if committed is None:
                    w, w_off = p, (u + slack) * p
                else:
                    if up >= 0:
                        had, had_off = demands[up] + bids[b, h, up], demand_offs[up] + bids_off[b, h, up]
                    else:
                        had = torch.zeros(length + nodes, dtype=torch.float64, device=q.device)
                        had[:length] = committed[b, h, :length].double()
                        had_off = torch.zeros_like(had)
                    demands.append(had)
                    demand_offs.append(had_off + 2.0 ** -23 * had)
                    den = had[at] + p + EPS
                    share = p / den
                    # d share = (dp had - p d had) / den^2, and the quotient's own 2^-21
                    share_off = (slack * p * had[at] + p * demand_offs[x][at]) / den ** 2 + 2.0 ** -20 * share
                    total = share.sum() + EPS
                    w = share / total
                    w_off = share_off / total + w * (share_off.sum() / total) + u * w
                o = w @ vals[at]
                out[b, h, x] = o
                off[b, h, x] = w_off @ vals[at].abs() + u * o.abs()
    return out, off, bids, bids_off


def evicted(scores, keep, recent, sinks):
    """(B, H, keep) positions that stay; a plain sort of (rank, position) pairs."""
    batch, heads, length = scores.shape
    index = torch.empty(batch, heads, keep, dtype=torch.int64)
    for b in range(batch):
        for h in range(heads):
            row = scores[b, h].tolist()
            held = set(range(sinks)) | set(range(length - recent, length))
            rest = sorted((x for x in range(length) if x not in held),
                          key=lambda x: (0 if row[x] != row[x] else 1, 0 if row[x] != row[x] else -row[x], x))
            index[b, h] = torch.tensor(sorted(held | set(rest[:keep - len(held)])))
    return index
