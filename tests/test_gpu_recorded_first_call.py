"""A thread whose first call of the library is recorded into a CUDA graph: the dilution operator on the tensor cores, forward and backward."""

from __future__ import annotations

import threading

import pytest
import torch

from conftest import load_package, make_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_a_thread_whose_first_call_is_recorded(dim):
    lib = load_package()
    q, k, v, dout = (x.cuda().to(torch.bfloat16) for x in make_inputs(1, 2, 200, dim, seed=3))

    def step(leaves):
        out = lib.dilution_attention(*leaves, dot_precision="bf16")
        return (out, *torch.autograd.grad(out, leaves, dout.to(out.dtype)))

    want = step([x.clone().requires_grad_(True) for x in (q, k, v)])
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    got, graph = [], torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def record():
        with torch.cuda.graph(graph):
            got.extend(step(leaves))

    thread = threading.Thread(target=record)
    thread.start()
    thread.join()
    graph.replay()
    torch.cuda.synchronize()
    assert len(got) == 4
    # (the operator adds its gradients in no fixed order: two fp32 sums of 200 terms, 200 2^-24 of the largest terms apart, may round to
    # neighbouring bf16 values, which are two half steps of 2^-8 apart)
    for a, b in zip(want, got):
        a, b = a.double(), b.double()
        assert ((a - b).abs() <= 2 ** -7 * a.abs() + 2 ** -14 * a.abs().max()).all()
