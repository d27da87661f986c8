"""What softmax_attention, tree steps and evict_cache refuse, before anything is launched (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import load_package

ONE = ctypes.c_void_p(256)          # never dereferenced: validation fails first
ODD = ctypes.c_void_p(264)


class OnCuda(torch.Tensor):
    """A host tensor that says it is on a CUDA device: the checks run, and what they let through would fail to launch."""
    is_cuda = property(lambda self: True)


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnCuda)


def message(rc):
    return load_package()._lib.load().dilution_last_error().decode() if rc else ""


def attend(dtype=1, batch=1, heads=2, kv=2, t=8, d=64, scale=0.125, cap=0.0, q=ONE, docs=None, ranges=None, out=ONE):
    lib = load_package()._lib.load()
    return lib.dilution_attend_forward(q, ONE, ONE, dtype, batch, heads, kv, t, d, scale, cap, None, docs, None, ranges, out, None, None, None)


@pytest.mark.parametrize("change,rc,text", [
    (dict(dtype=2), 1, "dtype"), (dict(d=48), 2, "head_dim"), (dict(heads=3), 1, "kv_heads"), (dict(t=0), 1, "sizes"),
    (dict(batch=0), 1, "sizes"), (dict(t=(1 << 30) + 1), 1, "grid"), (dict(t=1 << 40), 1, "sizes"), (dict(cap=-1.0), 1, "cap"),
    (dict(cap=float("inf")), 1, "cap"), (dict(cap=float("nan")), 1, "cap"), (dict(scale=0.0), 1, "scale"), (dict(q=None), 1, "null"),
    (dict(docs=ONE), 1, "null"), (dict(q=ODD), 1, "aligned"), (dict(batch=1 << 20, heads=64, kv=64, t=1 << 20), 1, "grid")])
def test_attend_forward(change, rc, text):
    got = attend(**change)
    assert got == rc and text in message(got)


def test_attend_backward():
    lib = load_package()._lib.load()
    args = [ONE, ONE, ONE, 1, 1, 2, 2, 8, 64, 0.125, 0.0, None, None, None, None, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, None]
    for at in (17, 18, 19, 20, 21, 22):
        rc = lib.dilution_attend_backward(*args[:at], None, *args[at + 1:])
        assert rc == 1 and "null" in message(rc)


def tree(fn="dilution_tree_softmax", dtype=1, batch=1, heads=2, group=1, nodes=4, cap=64, length=10, d=64, scale=0.125, softcap=0.0,
         q=ONE, scratch=ONE):
    lib = load_package()._lib.load()
    if fn == "dilution_tree_softmax":
        return lib.dilution_tree_softmax(q, ONE, ONE, ONE, ONE, dtype, batch, heads, group, nodes, cap, length, None, d, scale, softcap,
                                         None, ONE, 0, ONE, ONE, scratch, None)
    return lib.dilution_tree_dilute(q, ONE, ONE, ONE, ONE, dtype, batch, heads, nodes, cap, length, None, d, scale, 1e-9, ONE, ONE, 0, ONE,
                                    ONE, scratch, None)


@pytest.mark.parametrize("fn", ["dilution_tree_softmax", "dilution_tree_dilute"])
@pytest.mark.parametrize("change,rc,text", [
    (dict(dtype=7), 1, "dtype"), (dict(d=96), 2, "head_dim"), (dict(nodes=0), 1, "nodes"), (dict(nodes=65), 1, "nodes"),
    (dict(length=65), 1, "capacity"), (dict(length=-1), 1, "capacity"), (dict(batch=70000), 1, "batch"), (dict(q=None), 1, "null"),
    (dict(q=ODD), 1, "aligned"), (dict(scratch=None), 1, "null"), (dict(scratch=ODD), 1, "misaligned"), (dict(scale=-1.0), 1, "scale")])
def test_tree_steps(fn, change, rc, text):
    got = tree(fn, **change)
    assert got == rc and text in message(got)


def test_tree_accept():
    lib = load_package()._lib.load()

    def call(accepted=2, length=10, path=ONE, committed=ONE, advanced=ONE):
        return lib.dilution_tree_accept(ONE, ONE, ONE, ONE, ONE, 1, 1, 2, 1, 4, 12, length, None, 64, 0.125, 0.0, None, ONE, 0, ONE, path,
                                        0, accepted, committed, advanced, None)

    for change, text in ((dict(accepted=0), "accepted"), (dict(accepted=5), "accepted"), (dict(accepted=3), "accepted"),
                         (dict(path=None), "null"), (dict(advanced=None), "null"), (dict(committed=None), "null"),
                         (dict(length=13), "capacity")):
        rc = call(**change)
        assert rc == 1 and text in message(rc)


def test_evict():
    lib = load_package()._lib.load()

    def call(dtype=1, n=2, cap=64, length=40, d=64, stride=64, keep=10, recent=2, sinks=2, new=32, k=ONE, com=ONE, com_out=ONE):
        return lib.dilution_evict(k, ONE, com, dtype, n, cap, length, d, ONE, stride, keep, recent, sinks, new, ONE, ONE, com_out, ONE, None)

    for change, rc, text in ((dict(dtype=3), 1, "dtype"), (dict(d=24), 2, "head_dim"), (dict(length=0), 1, "length"),
                             (dict(length=65), 1, "length"), (dict(stride=39), 1, "length"), (dict(keep=0), 1, "keep"),
                             (dict(keep=41), 1, "keep"), (dict(recent=9), 1, "keep"), (dict(sinks=-1), 1, "keep"),
                             (dict(new=9), 1, "capacity"), (dict(k=None), 1, "null"), (dict(k=ODD), 1, "aligned"),
                             (dict(com=None), 1, "null"), (dict(com_out=None), 1, "null")):
        got = call(**change)
        assert got == rc and text in message(got), change


def test_sizes_of_scratch():
    lib = load_package()._lib.load()
    assert lib.dilution_attend_ranges_bytes(2, 65) == 2 * 2 * 16 and lib.dilution_attend_ranges_bytes(0, 5) == 0
    sizes = [lib.dilution_tree_scratch_bytes(2, 4, 2, 8, n, 64) for n in (0, 100, 10000)]
    assert 0 < sizes[0] <= sizes[1] <= sizes[2]
    assert lib.dilution_tree_scratch_bytes(2, 4, 0, 8, 100, 64) == 0


def test_softmax_attention_arguments():
    lib = load_package()
    q, k = fake(1, 4, 8, 64), fake(1, 2, 8, 64)
    run = lib.softmax_attention
    with pytest.raises(RuntimeError, match="CUDA"):
        run(torch.zeros(1, 4, 8, 64), torch.zeros(1, 2, 8, 64), torch.zeros(1, 2, 8, 64))
    for args in ((q, fake(1, 3, 8, 64), fake(1, 3, 8, 64)), (q, k, fake(1, 2, 9, 64)), (q, fake(1, 2, 9, 64), fake(1, 2, 9, 64)),
                 (q, fake(1, 2, 8, 64, dtype=torch.float32), k), (fake(1, 4, 8, 48), fake(1, 2, 8, 48), fake(1, 2, 8, 48)),
                 (fake(1, 4, 8, 64, dtype=torch.float16),) + (fake(1, 2, 8, 64, dtype=torch.float16),) * 2, (fake(4, 8, 64), k, k)):
        with pytest.raises(ValueError):
            run(*args)
    for options in (dict(softcap=0.0), dict(softcap=-3), dict(softcap=float("nan")), dict(slopes=torch.zeros(3)),
                    dict(slopes=torch.zeros(4, requires_grad=True)), dict(slopes=torch.zeros(4, dtype=torch.int32)),
                    dict(documents=torch.zeros(1, 8)), dict(documents=torch.zeros(1, 9, dtype=torch.int32)),
                    dict(documents=[0] * 8), dict(prefix=torch.zeros(2, dtype=torch.int32)), dict(prefix=torch.zeros(1))):
        with pytest.raises(ValueError):
            run(q, k, k, **options)


def caches(batch=1, heads=2, cap=16, dim=64, length=8, dtype=torch.bfloat16, **more):
    return dict(k=fake(batch, heads, cap, dim, dtype=dtype), v=fake(batch, heads, cap, dim, dtype=dtype), len=length, **more)


def test_tree_step_arguments():
    lib = load_package()
    q, k = fake(1, 4, 3, 64), fake(1, 2, 3, 64)
    step = lib.softmax_tree_step
    with pytest.raises(RuntimeError, match="CUDA"):
        step(torch.zeros(1, 4, 3, 64), torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3, 64), caches(), [-1, 0, 1])
    for parents in ([-1, 0], [-1, 1, 0], [-2, 0, 1], [[-1, 0, 1], [-1, 0, 1]], [0, 0, 0], torch.zeros(3), [-1.0, 0.0, 1.0]):
        with pytest.raises(ValueError):
            step(q, k, k, caches(), parents)
    for cache in (caches(heads=4), caches(dim=32), caches(length=17), caches(length=-1), caches(dtype=torch.float32), caches(batch=2)):
        with pytest.raises(ValueError):
            step(q, k, k, cache, [-1, 0, 1])
    with pytest.raises(ValueError, match="64 nodes"):
        step(fake(1, 2, 65, 64), fake(1, 2, 65, 64), fake(1, 2, 65, 64), caches(), list(range(-1, 64)))
    with pytest.raises(ValueError, match="softcap"):
        step(q, k, k, caches(), [-1, 0, 1], softcap=0)
    with pytest.raises(ValueError, match="key heads"):
        lib.dilution_tree_step(q, k, k, caches(committed=torch.zeros(1, 2, 16)), [-1, 0, 1])
    q = fake(1, 2, 3, 64)
    for demand in (torch.zeros(1, 2, 15), torch.zeros(1, 2, 16, dtype=torch.float64), torch.zeros(1, 16, 2).transpose(1, 2)):
        with pytest.raises(ValueError, match="committed"):
            lib.dilution_tree_step(q, k, k, caches(committed=demand), [-1, 0, 1])


def test_tree_accept_arguments():
    lib = load_package()
    draft = dict(q=fake(1, 2, 3, 64), k=fake(1, 2, 3, 64), v=fake(1, 2, 3, 64), tree=[-1, 0, 0], len=8)
    for cache, path in ((caches(), [0, 1, 2]), (caches(), [1]), (caches(), [0, 3]), (caches(), [-1]), (caches(length=9), [0]),
                        (caches(cap=9), [0, 1]), (caches(), [0, 1, 2, 2])):
        with pytest.raises(ValueError):
            lib.tree_accept(cache, draft, path)
    with pytest.raises(ValueError, match="no demand"):
        lib.tree_accept(caches(), draft, [0], out=torch.zeros(1, 2, 16))
    with pytest.raises(ValueError, match="out"):
        lib.tree_accept(caches(committed=torch.zeros(1, 2, 16)), draft, [0], out=torch.zeros(1, 2, 15))
    with pytest.raises(ValueError):
        lib.tree_accept(caches(), dict(draft, tree=None), [3])
    # nothing accepted: nothing moves
    cache = caches(committed=torch.ones(1, 2, 16))
    out = torch.zeros(1, 2, 16)
    assert lib.tree_accept(cache, draft, [], out=out) is out and cache["len"] == 8
    assert (out[:, :, :8] == 1).all() and (out[:, :, 8:] == 0).all()


def test_evict_arguments():
    lib = load_package()
    with pytest.raises(RuntimeError, match="CUDA"):
        lib.evict_cache(dict(k=torch.zeros(1, 2, 16, 64), v=torch.zeros(1, 2, 16, 64), len=8), 4)
    demand = torch.zeros(1, 2, 16)
    for keep, more in ((0, {}), (9, {}), (4, dict(recent=5)), (4, dict(recent=2, sinks=3)), (4, dict(recent=-1)), (4, dict(capacity=3)),
                       (4, dict(scores=torch.zeros(1, 2, 7))), (4, dict(scores=torch.zeros(1, 3, 8))),
                       (4, dict(scores=torch.zeros(1, 2, 8, dtype=torch.float64)))):
        with pytest.raises(ValueError):
            lib.evict_cache(caches(committed=demand), keep, **more)
    with pytest.raises(ValueError, match="needs scores"):
        lib.evict_cache(caches(), 4)
    with pytest.raises(ValueError, match="device"):
        lib.evict_cache(caches(committed=demand, pos_dev=torch.zeros(1, dtype=torch.int32)), 4)


def test_a_recorded_decode_refuses_evicted_caches_of_rotated_layers():
    from types import SimpleNamespace
    lib = load_package()
    model = SimpleNamespace(config=SimpleNamespace(positional="rope"))
    with pytest.raises(ValueError, match="evicted"):
        lib.GraphedDecode(model, [caches(evicted=3)])


def test_rest_is_of_bf16_outputs():
    lib = load_package()._lib.load()
    rc = lib.dilution_attend_forward(ONE, ONE, ONE, 0, 1, 2, 2, 8, 64, 0.125, 0.0, None, None, None, None, ONE, ONE, None, None)
    assert rc == 1 and "rest" in message(rc)


def test_attend_sizes_whose_product_wraps():
    big = (1 << 31) - 1
    got = attend(batch=big, heads=big, kv=1, t=1 << 30)
    assert got == 1 and "grid" in message(got)


def test_slopes_over_an_evicted_cache():
    lib = load_package()
    q, k = fake(1, 4, 3, 64), fake(1, 2, 3, 64)
    with pytest.raises(ValueError, match="evicted"):
        lib.softmax_tree_step(q, k, k, caches(evicted=2), [-1, 0, 1], slopes=torch.zeros(4))


def test_a_dilution_step_needs_the_demand():
    q = fake(1, 2, 3, 64)
    with pytest.raises(ValueError, match="committed"):
        load_package().dilution_tree_step(q, q, q, caches(), [-1, 0, 1])


class Rotated:
    """A layer of the model as far as the cached steps ask."""
    rope, d_model, n_heads = object(), 128, 2

    def __init__(self, fast):
        self.fast = fast

    def _kernel_ok(self, x):
        return self.fast

    def _standard(self):
        return True

    def _split_heads(self, x, offset):
        raise StopIteration(offset)

    def _unfused_step_cache(self, x, cache):
        raise LookupError

    _b200_step_cache = _unfused_step_cache


@pytest.mark.parametrize("name,fused", [("kernels", "_fused_step_cache"), ("layers", "_softmax_step_cache")])
def test_cached_steps_rotate_by_the_tokens_that_there_have_been(name, fused):
    step = getattr(getattr(load_package(), name), fused)
    for evicted, offset in ((0, 8), (5, 13)):
        with pytest.raises(StopIteration) as stop:
            step(Rotated(True), fake(1, 1, 128), caches(evicted=evicted))
        assert stop.value.args == (offset,)
    # a layer whose own step runs instead: it would rotate by the cache's length
    with pytest.raises(ValueError, match="evicted"):
        step(Rotated(False), torch.zeros(1, 1, 128), caches(evicted=5))
    with pytest.raises(LookupError):
        step(Rotated(False), torch.zeros(1, 1, 128), caches())
