"""What the rounding of out to bf16 leaves off reaches the gradients on the tensor cores: values far from zero and next to one another, so
that dout . (v - out) is small next to dout . out.  Queries of zeros: every weight is 1 / n and its bf16 form is exact."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package, seeded
from test_gpu_masked import DEV, call

pytestmark = pytest.mark.gpu


def uniform(seq, dim):
    q = torch.zeros(2, 4, seq, dim, device=DEV, dtype=torch.bfloat16)
    k = seeded((2, 2, seq, dim), 1).to(DEV, torch.bfloat16)
    v = (256 + 2 * (seeded((2, 2, seq, dim), 2) > 0)).to(DEV, torch.bfloat16)
    return q, k, v, seeded((2, 4, seq, dim), 3).to(DEV, torch.bfloat16)


def plain(q, k, v):
    q, k, v = q.double(), *(x.double().repeat_interleave(2, 1) for x in (k, v))
    seq = q.shape[2]
    p = torch.ones(seq, seq, device=DEV, dtype=torch.float64).tril()
    return k, v, (p / p.sum(-1, keepdim=True)).expand(2, 4, seq, seq)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq", [2, 3, 9, 65, 130])
def test_gradients_of_close_values(seq, dim):
    """dq is off by 2^-8 |ds| |k| for the rounding of dS, and by e = p (|dout| (v + out)) |k| times 2^-16 for the rounded rest (2^-8 of 2^-8)
    and 2^-16 for sums of at most 128 + 130 terms, 1 / n and its product (2^-24 each, half of it at random signs is not taken off)."""
    q, k, v, dout = x = uniform(seq, dim)
    _, dq, _, _ = call(x)
    k, v, p = plain(q, k, v)
    dout = dout.double()
    out = p @ v
    ds = p * (dout @ v.mT - (dout * out).sum(-1, keepdim=True))
    want = ds @ k / dim ** 0.5
    size = p * (dout.abs() @ v.abs().mT + (dout * out).abs().sum(-1, keepdim=True))
    off = (2 ** -8 * ds.abs() + (2 ** -16 + 2 ** -16) * size) @ k.abs() / dim ** 0.5
    assert ((dq.double() - want).abs() <= 2 ** -8 * want.abs() + off).all()


@pytest.mark.parametrize("dim", [16, 32, 64, 128])
def test_out_and_its_rest(dim):
    """out + rest, by the C entry: 2^-16 for the rounded rest, (130 + 8) 2^-24 for the sums and the division."""
    lib = load_package()._lib
    seq = 130
    q, k, v, _ = uniform(seq, dim)
    out, rest = torch.empty_like(q), torch.empty_like(q)
    lib.check(lib.load().dilution_attend_forward(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), lib.BF16, 2, 4, 2, seq, dim, dim ** -0.5, 0.0, None, None, None, None, out.data_ptr(),
        rest.data_ptr(), None, torch.cuda.current_stream().cuda_stream), "forward")
    _, v, p = plain(q, k, v)
    want = p @ v
    assert ((out.double() + rest.double() - want).abs() <= (2 ** -16 + 138 * 2 ** -24) * want).all()
    assert (rest != 0).any()
