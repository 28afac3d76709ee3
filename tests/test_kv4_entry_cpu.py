"""Who sees the ops of the 4-bit cache by name: the calls go straight to the binding only with plain tensors and
nothing that maps or watches them. The binding is replaced here by one that takes notes."""
import types

import pytest
import torch

from vllm_sly_radiance_amd import radiance_kv4 as K


def q_k(n=3):
    return (torch.arange(n * 2 * 64, dtype=torch.float32).view(n, 2, 64).to(torch.bfloat16),
            torch.ones((n, 1, 64), dtype=torch.bfloat16))


@pytest.fixture
def seen(monkeypatch):
    """The arguments of each call that reached the binding."""
    calls, is_plain, fake = [], K._native.ops().is_plain, types.SimpleNamespace()

    def note(name, out):
        def op(*args):
            for a in args:
                if isinstance(a, torch.Tensor):
                    assert type(a) in (torch.Tensor, torch.nn.Parameter)
                    assert not torch._C._functorch.is_functorch_wrapped_tensor(a)
                    a.data_ptr()
            calls.append(args)
            return out(*args)
        setattr(fake, name, op)
        setattr(fake, name + "_if_plain", lambda *a: op(*a) if is_plain(*a) else NotImplemented)
    note("qk_norm_rope", lambda q, k, *_: (q * 2, k * 3))
    note("gather", lambda cache, slots: (slots.to(torch.bfloat16), -slots.to(torch.bfloat16)))
    note("attention", lambda q, *_: q + 1)
    note("move_pages", lambda *_: None)
    monkeypatch.setattr(K._native, "ops", lambda: fake)
    return calls


def test_plain_tensors_take_the_short_way(seen):
    from torch.utils._python_dispatch import TorchDispatchMode
    q, k = q_k()
    a, b = K.qk_norm_rope(q, k, torch.nn.Parameter(q[0, 0], requires_grad=False), None, None, None)
    assert torch.equal(a, q * 2) and torch.equal(b, k * 3) and seen[0][0] is q

    ops = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            ops.append(str(func))
            return func(*args, **(kwargs or {}))
    with Watch():
        K.attention(q, torch.zeros((1, 1, 1, 17 * 64), dtype=torch.uint8), torch.zeros((1, 1), dtype=torch.int32),
                    torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1, 1)
    assert "radiance.kv4_attention.default" in ops


def test_vmap_maps(seen):
    """Each slice reaches the binding as a plain tensor."""
    q = torch.stack([q_k()[0] * i for i in range(4)])
    k = torch.stack([q_k()[1] * i for i in range(4)])
    a, b = torch.func.vmap(lambda q, k: K.qk_norm_rope(q, k, None, None, None, None))(q, k)
    assert torch.equal(a, q * 2) and torch.equal(b, k * 3) and len(seen) == 4
    # mapped over an argument that is not the first
    seen.clear()
    cache = torch.zeros((1, 1, 1, 17 * 64), dtype=torch.uint8)
    slots = torch.arange(6).view(2, 3)
    a, b = torch.func.vmap(lambda s: K.gather(cache, s))(slots)
    assert torch.equal(a, slots.to(torch.bfloat16)) and torch.equal(b, -a) and len(seen) == 2


class Marked(torch.Tensor):
    names = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.names.append(str(func))
        with torch._C.DisableTorchFunctionSubclass():
            return func(*(a.as_subclass(torch.Tensor) if isinstance(a, Marked) else a for a in args),
                        **(kwargs or {}))


@pytest.mark.parametrize("which", [0, 1, 2])
def test_subclasses_see_the_op(seen, which):
    args = [*q_k(), q_k()[0][0, 0]]
    args[which] = args[which].as_subclass(Marked)
    Marked.names.clear()
    K.qk_norm_rope(args[0], args[1], args[2], None, None, None)
    assert any("qk_norm_rope" in n for n in Marked.names) and len(seen) == 1
    Marked.names.clear()
    K.move_pages(torch.zeros((1, 1, 1, 17 * 64), dtype=torch.uint8), torch.zeros((0, 2), dtype=torch.int32),
                 torch.zeros((1, 1), dtype=torch.int32).as_subclass(Marked))
    assert any("kv4_move_pages" in n for n in Marked.names)


def test_torch_func_grad_is_refused(seen):
    q, k = (x.float() for x in q_k())
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda q: K.qk_norm_rope(q, k, None, None, None, None)[0].sum())(q)


def test_what_is_plain():
    is_plain = K._native.ops().is_plain
    t = torch.zeros(3)
    assert is_plain() and is_plain(None, 3, 2.5, True, t, torch.nn.Parameter(t, requires_grad=False), [t], "x")
    asks = torch.zeros(3, requires_grad=True)
    assert not is_plain(t, asks) and not is_plain(t.as_subclass(Marked)) and is_plain(asks.detach())
    with torch.no_grad():
        assert is_plain(t, asks)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = mode.from_tensor(t)
    assert not is_plain(fake)
    assert not is_plain(torch._to_functional_tensor(t))
    torch.func.vmap(lambda x: (is_plain(x) and pytest.fail("a batched tensor")) or x * 2)(torch.zeros(2, 2))
    torch.func.grad(lambda x: (is_plain(x) and pytest.fail("a tensor under grad")) or x.sum())(t)
    torch.func.jvp(lambda x: (is_plain(x) and pytest.fail("a tensor under jvp")) or x * 2, (t,), (t,))


def test_views_that_are_not_their_bytes_are_not_plain():
    """A negated view, or a tensor of zeros without memory: the dispatcher makes plain ones of them."""
    is_plain = K._native.ops().is_plain
    t = torch.arange(3.0)
    assert not is_plain(torch._neg_view(t)) and not is_plain(torch._efficientzerotensor((3,)))
    assert is_plain(torch._neg_view(t).resolve_neg(), t[::2], t.expand(2, 3))


def test_a_negated_view_is_what_it_says(seen):
    q, k = q_k()
    a, b = K.qk_norm_rope(torch._neg_view(q), k, None, None, None, None)
    assert torch.equal(a, -2 * q) and torch.equal(b, 3 * k)
    assert not seen[0][0].is_neg()
