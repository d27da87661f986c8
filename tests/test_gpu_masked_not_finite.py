"""Values that are not finite in softmax_attention: what they reach is what the formula says, and no call takes long over them."""

from __future__ import annotations

import pytest
import torch

from oracle import operators_oracle as O
from test_gpu_masked import DEV, TYPES, call, inputs

pytestmark = pytest.mark.gpu


def formula(q, k, v, dout, documents, prefix=None):
    """Which elements of (out, dq, dk, dv) are finite: sums over the pairs that see one another alone, term by term in 64 bits."""
    heads, seq, dim = q.shape[1:]
    group = heads // k.shape[1]
    see = O.visible(seq, documents, prefix, q.device)
    got = [torch.zeros(x.shape, device=DEV, dtype=torch.float64) for x in (q, q, k, k)]
    add = lambda w, x: torch.where(see[..., None], w[..., None] * x, 0.0)
    for h in range(heads):
        qs, do, ks, vs = (x[0, at].double() for x, at in ((q, h), (dout, h), (k, h // group), (v, h // group)))
        z = (qs[:, None] * ks[None]).sum(-1) * dim ** -0.5
        z = z.masked_fill(~see, -torch.inf)
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(top == -torch.inf, 0.0, top)).masked_fill(~see, 0.0)
        mass = e.sum(-1, keepdim=True)
        p = e / torch.where(mass == 0, 1.0, mass)
        out = add(p, vs[None]).sum(1)
        ds = p * ((do[:, None] * vs[None]).sum(-1) - (do * out).sum(-1, keepdim=True))
        got[0][0, h] = out
        got[1][0, h] = add(ds, ks[None]).sum(1)
        got[2][0, h // group] += add(ds, qs[:, None]).sum(0)
        got[3][0, h // group] += add(p, do[:, None]).sum(0)
    return [torch.isfinite(x) for x in got]


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("where", [0, 1, 2, 3])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("at,feature,docs", [(0, slice(None), 0), (70, 3, 0), (149, 1, 0), (slice(None), 5, 0), (70, slice(None), 40),
                                            (slice(60, 90), 2, 7), (slice(None), slice(None), 50)])
def test_what_they_reach(at, feature, docs, value, where, dtype, dim):
    x = list(inputs(1, 2, 1, 150, dim, dtype))
    documents = (torch.arange(150, device=DEV) // docs)[None].contiguous() if docs else None
    want, off = O.attention(*x, documents=documents)
    x[where] = x[where].clone()
    x[where][:, :, at, feature] = value
    got = call(x, documents=documents)
    for name, a, b, far, finite in zip(("out", "dq", "dk", "dv"), got, want, off, formula(*x, documents[0] if docs else None)):
        assert torch.equal(torch.isfinite(a), finite), name
        # (numbers where the formula has them are those of finite inputs, if the weights have not moved: q and k that are infinite
        # take part in rows whose scores are all -inf)
        if where in (2, 3) or value != value:
            assert ((a.double() - b).abs() <= far + 1e-12)[finite].all(), name


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("where", [0, 1, 2, 3])
@pytest.mark.parametrize("at,feature", [(0, slice(None)), (69, 3), (70, slice(None)), (140, 1), (200, slice(None)), (slice(90, 210), 5)])
@pytest.mark.parametrize("docs", [0, 90])
def test_over_a_prefix(docs, at, feature, where, dtype, dim):
    """Keys in front of the prefix's end have queries of other tiles behind them that see them, and later keys of their tile do not."""
    x = list(inputs(1, 2, 1, 210, dim, dtype))
    documents = (torch.arange(210, device=DEV) // docs)[None].contiguous() if docs else None
    prefix = torch.tensor([70], device=DEV)
    want, off = O.attention(*x, documents=documents, prefix=prefix)
    x[where] = x[where].clone()
    x[where][:, :, at, feature] = float("nan")
    got = call(x, documents=documents, prefix=prefix)
    for name, a, b, far, finite in zip(("out", "dq", "dk", "dv"), got, want, off, formula(*x, documents[0] if docs else None, 70)):
        assert torch.equal(torch.isfinite(a), finite), name
        assert ((a.double() - b).abs() <= far + 1e-12)[finite].all(), name


def took(x, documents=None):
    call(x, documents=documents)
    times = []
    for _ in range(3):
        start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        call(x, documents=documents)
        stop.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(stop))
    return min(times)


@pytest.mark.parametrize("dtype,seq", [(torch.bfloat16, 4096), (torch.float32, 1024)])
@pytest.mark.parametrize("docs", [0, 3])
def test_they_take_no_long_time(docs, dtype, seq):
    """A NaN in an early key or in all of dout makes every row no number by right, one in a query or of padding no row that was one.  None
    takes 25 times as long as finite values do (up to 220 times where every such row is walked through).  Documents that
    interleave token by token have a token of another document in every tile: their rows are walked through, 32 by each warp of a CTA of
    four in each of three kernels, where a pair takes a warp less than 0.15 us."""
    x = inputs(1, 4, 4, seq, 64, dtype)
    documents = (torch.arange(seq, device=DEV) % docs)[None].contiguous() if docs else None
    limit = 25 * took(x, documents) + (3 * 32 * seq * 0.15e-3 if docs else 0)
    for where, at in ((1, 0), (1, seq // 2), (3, slice(None)), (3, seq - 1), (0, seq // 2), (2, seq // 2)):
        y = [t.clone() for t in x]
        y[where][:, :, at] = float("nan")
        assert took(y, documents) <= limit, (where, at)
    lone = torch.zeros(1, seq, device=DEV, dtype=torch.int64) if documents is None else documents.clone()
    lone[:, seq - 100] = -1
    y = [t.clone() for t in x]
    for t in y:
        t[:, :, seq - 100] = float("nan")
    assert took(y, lone) <= limit


@pytest.mark.parametrize("dtype,dim,seq", [*((*t, 333) for t in TYPES), (torch.bfloat16, 64, 270000), (torch.bfloat16, 128, 270000)])
def test_padding_changes_no_bit(dtype, dim, seq):
    """Padding at the end and inside tiles, of finite values and of NaN (270000 tokens are more than a block keeps notes of)."""
    x = inputs(1, 2, 1, seq, dim, dtype)
    at = torch.arange(seq, device=DEV)
    documents = torch.where((at % 450 >= 447) | (at % 97 == 5) | (at >= seq - 30), -1, at // 450)[None].contiguous()
    want = call(x, documents=documents)
    y = [t.clone() for t in x]
    for t in y:
        t[:, :, documents[0] < 0] = float("nan")
    assert all(torch.equal(a, b) for a, b in zip(want, call(y, documents=documents)))
