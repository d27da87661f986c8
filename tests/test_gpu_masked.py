"""softmax_attention: capped scores, distance bias, documents and prefixes, forward and backward, against the formulas in 64
bits.  Every bound is element by element and counts roundings (oracle/operators_oracle.py)."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package, seeded
from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(batch, heads, kv_heads, seq, dim, dtype, seed=0, q_scale=1.0):
    q = seeded((batch, heads, seq, dim), seed, q_scale).to(DEV, dtype)
    k, v = (seeded((batch, kv_heads, seq, dim), seed + s).to(DEV, dtype) for s in (1, 2))
    return q, k, v, seeded((batch, heads, seq, dim), seed + 3, 1e-1).to(DEV, dtype)


def documents_of(batch, seq, mean, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    rows = torch.zeros(batch, seq, dtype=torch.int64)
    for b in range(batch):
        at, doc = 0, 3
        while at < seq:
            n = int(torch.randint(1, 2 * mean, (1,), generator=g))
            rows[b, at:at + n] = doc
            at, doc = at + n, doc + 1
        if pad:
            rows[b, seq - pad * (b + 1):] = -1
    return rows.to(DEV)


def call(x, **options):
    q, k, v, dout = x
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = load_package().softmax_attention(*leaves, **options)
    assert out.dtype == q.dtype and out.shape == q.shape
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def check(x, **options):
    got = call(x, **options)
    want, off = O.attention(*x, **options)
    for name, a, b, far in zip(("out", "dq", "dk", "dv"), got, want, off):
        assert torch.isfinite(a).all(), name
        worst = ((a.double() - b).abs() - far).max().item()
        assert worst <= 1e-12, (name, worst, (a.double() - b).abs().max().item())
    # without gradients: the same forward
    with torch.no_grad():
        assert torch.equal(load_package().softmax_attention(*x[:3], **options), got[0])
    return got


TYPES = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 32),
         (torch.float32, 16)]


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("seq", [1, 2, 63, 64, 65, 127, 128, 129, 200, 257, 391])
def test_causal_lengths(seq, dtype, dim):
    check(inputs(1, 2, 2, seq, dim, dtype))


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [2.0, 30.0])
def test_capped_scores(cap, dtype, dim):
    check(inputs(1, 2, 1, 210, dim, dtype, q_scale=3.0), softcap=cap)


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_distance_bias(dtype, dim):
    slopes = torch.tensor([0.5, 2.0 ** -6, 0.0], device=DEV)
    check(inputs(2, 3, 3, 300, dim, dtype), slopes=slopes)


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("mean,pad", [(3, 0), (40, 7), (150, 70), (1000, 0)])
def test_documents(mean, pad, dtype, dim):
    docs = documents_of(2, 330, mean, seed=mean, pad=pad)
    got = check(inputs(2, 2, 2, 330, dim, dtype), documents=docs)
    for x in got:
        assert (x.transpose(1, 2)[docs < 0] == 0).all()      # padding: nothing out, no gradients


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("prefix", [0, 1, 64, 100, 129, 270, 9999])
def test_prefix(prefix, dtype, dim):
    check(inputs(2, 2, 1, 270, dim, dtype), prefix=torch.tensor([prefix, prefix // 3], device=DEV))


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_everything_at_once(dtype, dim):
    check(inputs(2, 4, 2, 391, dim, dtype, q_scale=2.0), softcap=15.0, slopes=torch.tensor([0.3, 0.1, 0.03, 0.01], device=DEV),
          documents=documents_of(2, 391, 90, seed=5, pad=20), prefix=torch.tensor([150, 77], device=DEV, dtype=torch.int32))


@pytest.mark.parametrize("heads,kv_heads", [(6, 1), (6, 2), (8, 8)])
@pytest.mark.parametrize("dtype,dim", TYPES[:3])
def test_heads_that_share_keys(dtype, dim, heads, kv_heads):
    check(inputs(2, heads, kv_heads, 150, dim, dtype))


@pytest.mark.parametrize("dim", [16, 32])
@pytest.mark.parametrize("seq", [1, 2, 7])
def test_few_keys_and_the_rounding_of_out(seq, dim):
    """ds = p (dout . v - delta) is a difference; delta is of out before its rounding to bf16.  Off by, next to terms of size
    e = sum_d |dout_d| (|v_jd| + |out_d|): 2^-16 e for the rounded rest of out (2^-8 of 2^-8), 2^-18 e for 32-bit sums of up to
    32 + 7 terms and the exponential; and dq's own rounding, 2^-8 of it."""
    q, k, v, dout = x = inputs(4, 8, 8, seq, dim, torch.bfloat16, seed=11)
    _, dq, _, _ = call(x)
    q, k, v, dout = (t.double() for t in x)
    p = (q @ k.mT / dim ** 0.5).masked_fill(torch.ones(seq, seq, device=DEV).tril() == 0, -torch.inf).softmax(-1)
    out = p @ v
    want = p * (dout @ v.mT - (dout * out).sum(-1, keepdim=True)) @ k / dim ** 0.5
    size = p * (dout.abs() @ v.abs().mT + (dout * out).abs().sum(-1, keepdim=True)) @ k.abs() / dim ** 0.5
    assert ((dq.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -16 + 2 ** -18) * size).all()


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_long_rows(dtype, dim):
    check(inputs(1, 2, 1, 2100, dim, dtype), documents=documents_of(1, 2100, 700, seed=9))


@pytest.mark.parametrize("dim", [64, 128])
def test_more_half_tiles_than_a_block_keeps_notes_of(dim):
    """270000 tokens, which are over 4096 half tiles of keys, in documents of 450: the first and the last ones as rows of their own."""
    seq, doc, near = 270000, 450, 8
    docs = (torch.arange(seq, device=DEV) // doc).expand(1, seq).contiguous()
    x = inputs(1, 2, 1, seq, dim, torch.bfloat16)
    got = call(x, documents=docs)
    for first in (0, seq // 2 // doc * doc, seq - near * doc):
        rows = [t[0, :, first:first + near * doc].unflatten(1, (near, doc)).transpose(0, 1) for t in (*x, *got)]
        want, off = O.attention(*rows[:4])
        for a, b, far in zip(rows[4:], want, off):
            assert ((a.double() - b).abs() <= far + 1e-12).all()


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
@pytest.mark.parametrize("std", [8.0, 40.0])
def test_peaked_scores(dtype, dim, std):
    """Scores of a large spread: the running maximum moves late and far."""
    x = inputs(1, 1, 1, 333, dim, dtype, q_scale=std)
    ramp = torch.linspace(0.2, 2.0, 333, device=DEV)[:, None]
    check((x[0], (x[1] * ramp).to(dtype), x[2], x[3]))


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_scores_that_grow_with_the_distance(dtype, dim):
    """By about 90 (in the exponent of 2) over 64 keys: whatever the order of the keys, the reference of a row moves many times."""
    q, k, v, dout = inputs(1, 2, 1, 700, dim, dtype)
    far = torch.arange(700, 0, -1, device=DEV)[:, None] * (dim ** -0.5 / 4)
    check(((q / 8 + 4).to(dtype), (k + far).to(dtype), v, dout))


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_ids_in_any_order(dtype, dim):
    """Documents that interleave: masks inside every tile."""
    docs = (torch.arange(260, device=DEV) % 3).expand(2, 260).contiguous()
    docs[1] = 5 - docs[1]
    check(inputs(2, 2, 2, 260, dim, dtype), documents=docs.to(torch.int32))


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_padding_may_hold_anything(dtype, dim, value):
    docs = documents_of(1, 200, 60, seed=2, pad=30)
    docs[0, 20:25] = -1
    x = inputs(1, 2, 2, 200, dim, dtype)
    for t in x:
        t[:, :, 20:25] = value
        t[:, :, 170:] = value
    check(x, documents=docs)


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("where", ["k", "v", "q", "dout"])
def test_a_later_token_that_is_not_finite(dtype, dim, where):
    """What a token may not see does not reach it: rows in front of a NaN key or value, keys behind a NaN query.  (Rows that are
    computed again add up in another order: they keep the formulas' bounds, not their bits.)"""
    at, which = 131, "qkv".index(where) if where in "qkv" else 3
    x = list(inputs(1, 1, 1, 200, dim, dtype))
    want, off = O.attention(*x)
    x[which] = x[which].clone()
    x[which][0, 0, at, 3] = float("nan")
    got = call(x)
    keep = torch.arange(200, device=DEV)
    keep = {"out": keep < at, "dq": keep < at, "dk": keep > at, "dv": keep > at} if where in "kv" else \
        {"out": keep != at, "dq": keep != at, "dk": keep > at, "dv": keep > at}
    for name, a, b, far in zip(("out", "dq", "dk", "dv"), got, want, off):
        if where in "kv" and name in ("dk", "dv"):
            continue                         # every query behind the key hands its NaN to all keys
        rows = keep[name]
        assert ((a[:, :, rows].double() - b[:, :, rows]).abs() <= far[:, :, rows] + 1e-12).all(), name
    if where in "kv":
        assert got[0][:, :, at:].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_slices(dtype):
    """(B, T, H, D) views, slices off a 16-byte boundary and an expanded upstream gradient."""
    b, h, t, d = 2, 3, 140, 64
    base = [seeded((b, t, h, d), s).to(DEV, dtype) for s in range(3)]
    q, k, v = (x.transpose(1, 2) for x in base)
    flat = seeded((b * h * t * d + 1,), 7).to(DEV, dtype)
    k = flat[1:].view(b, h, t, d)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    load_package().softmax_attention(*leaves).float().sum().backward()
    want, off = O.attention(q, k, v, torch.ones(1, device=DEV, dtype=dtype).expand(q.shape))
    for a, b_, far in zip((x.grad for x in leaves), want[1:], off[1:]):
        assert ((a.double() - b_).abs() <= far + 1e-12).all()


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_results_repeat(dtype, dim):
    x = inputs(2, 4, 2, 700, dim, dtype)
    docs = documents_of(2, 700, 200, seed=1)
    first = call(x, documents=docs)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call(x, documents=docs)))


def test_gradients_against_differences():
    """fp32, along random directions: (L(x + h e) - L(x - h e)) / 2 h with h^2 and the rounding of L in the bound."""
    x = inputs(1, 2, 1, 70, 32, torch.float32, q_scale=2.0)
    options = dict(softcap=8.0, slopes=torch.tensor([0.1, 0.02], device=DEV), documents=documents_of(1, 70, 30, seed=4))
    grads = call(x, **options)[1:]
    run = load_package().softmax_attention
    for at, g in enumerate(grads):
        e = seeded(x[at].shape, 50 + at).to(DEV)
        h = 1e-2

        def loss(sign):
            y = [t.clone() for t in x[:3]]
            y[at] = y[at] + sign * h * e
            return (run(*y, **options).double() * x[3].double()).sum().item()

        want = (loss(1) - loss(-1)) / (2 * h)
        got = (g.double() * e.double()).sum().item()
        # third derivatives of scores of about 2: some tens of h^2 |L|; rounding of L: 2^-22 |terms| / h
        size = (x[3].abs().sum().item()) * 2.0 ** -22 / h + 30 * h * h * abs(want) + 30 * h * h * g.norm().item()
        assert abs(got - want) <= size, (at, got, want, size)


def test_a_captured_call_is_replayed():
    x = inputs(1, 2, 2, 300, 64, torch.bfloat16)
    docs = documents_of(1, 300, 80, seed=3)
    static = [t.clone().requires_grad_(i < 3) for i, t in enumerate(x)]
    run = load_package().softmax_attention

    def step():
        out = run(*static[:3], documents=docs)
        return (out, *torch.autograd.grad(out, static[:3], static[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (20, 30):
        fresh = inputs(1, 2, 2, 300, 64, torch.bfloat16, seed=seed)
        other = documents_of(1, 300, 50, seed=seed)
        with torch.no_grad():
            for a, b in zip(static, fresh):
                a.copy_(b)
            docs.copy_(other)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, call(fresh, documents=other)))


def test_another_stream_and_two_calls_at_once():
    x, y = inputs(2, 4, 4, 600, 64, torch.bfloat16), inputs(2, 4, 4, 600, 64, torch.bfloat16, seed=40)
    want = [call(x), call(y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, t in zip(streams, (x, y)):
        with torch.cuda.stream(s):
            got.append(call(t))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_empty_calls():
    q = torch.zeros(2, 4, 0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    k = torch.zeros(2, 2, 0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out = load_package().softmax_attention(q, k, k)
    out.sum().backward()
    assert out.shape == q.shape and q.grad.shape == q.shape and k.grad.shape == k.shape


def test_a_thread_whose_first_call_is_recorded():
    """Forward and backward recorded by a thread that has made no call of the library before."""
    import threading
    x = inputs(1, 2, 2, 200, 64, torch.bfloat16)
    want, got, graph = call(x), [], torch.cuda.CUDAGraph()
    leaves = [t.detach().clone().requires_grad_(True) for t in x[:3]]
    torch.cuda.synchronize()

    def record():
        with torch.cuda.graph(graph):
            out = load_package().softmax_attention(*leaves)
            got.extend((out, *torch.autograd.grad(out, leaves, x[3])))

    thread = threading.Thread(target=record)
    thread.start()
    thread.join()
    graph.replay()
    torch.cuda.synchronize()
    assert len(got) == 4 and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dim", [32, 64])
def test_gradients_without_the_rest_of_out(dim):
    """The C entries with rest NULL: delta is of the rounded out, within the bounds that count that rounding."""
    lib = load_package()._lib
    q, k, v, dout = x = inputs(1, 2, 2, 150, dim, torch.bfloat16)
    out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse = torch.empty(1, 2, 150, device=DEV)
    scratch = torch.empty(lib.load().dilution_attend_scratch_bytes(1, 2, 150), device=DEV, dtype=torch.uint8)
    head = [q.data_ptr(), k.data_ptr(), v.data_ptr(), lib.BF16, 1, 2, 2, 150, dim, dim ** -0.5, 0.0, None, None, None, None]
    stream = torch.cuda.current_stream().cuda_stream
    lib.check(lib.load().dilution_attend_forward(*head, out.data_ptr(), None, lse.data_ptr(), stream), "forward")
    lib.check(lib.load().dilution_attend_backward(*head, out.data_ptr(), None, lse.data_ptr(), dout.data_ptr(), scratch.data_ptr(),
                                                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), stream), "backward")
    want, off = O.attention(*x)
    for a, b, far in zip((out, dq, dk, dv), want, off):
        assert ((a.double() - b).abs() <= far + 1e-12).all()
