"""Who sees the convolution, the delta rule and sampling by name: the calls go straight to the binding only with
plain tensors and nothing that maps or watches them. The binding is replaced here by one that takes notes."""
import types

import pytest
import torch

from vllm_sly_radiance_amd import radiance_gdn as G
from vllm_sly_radiance_amd import radiance_sample as S


@pytest.fixture
def seen(monkeypatch):
    """The arguments of each call that reached the binding."""
    calls, is_plain, fake = [], G._native.ops().is_plain, types.SimpleNamespace()

    def note(name, out):
        def op(*args):
            for a in args:
                if isinstance(a, torch.Tensor):
                    assert type(a) in (torch.Tensor, torch.nn.Parameter)
                    a.data_ptr()
            calls.append(args)
            return out(*args)
        setattr(fake, name, op)
        setattr(fake, name + "_if_plain", lambda *a: op(*a) if is_plain(*a) else NotImplemented)
    note("causal_conv", lambda x, *_: x + 1)
    note("gated_delta_rule", lambda q, k, v, *_: v + 1)
    note("sample", lambda x, *a: (torch.zeros(len(x), dtype=torch.int64), torch.zeros(len(x) if a[-1] else 0)))
    monkeypatch.setattr(G._native, "ops", lambda: fake)
    return calls


def batch(n):
    return torch.tensor([0, n], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), n


def conv_args(n=3):
    return (torch.ones((n, 16), dtype=torch.bfloat16), torch.ones((16, 4), dtype=torch.bfloat16), None,
            G.new_conv_state(2, 16, 4, "cpu"), *batch(n))


def delta_args(n=3):
    x = torch.ones((n, 2, 64), dtype=torch.bfloat16)
    g = torch.zeros((n, 2), dtype=torch.bfloat16)
    return (x, x, x, g, g, torch.zeros(2), torch.zeros(2), G.new_state(2, 2, 64, 64, "cpu"), *batch(n))


def test_plain_tensors_take_the_short_way(seen):
    from torch.utils._python_dispatch import TorchDispatchMode
    x = conv_args()
    assert G.causal_conv(*x).shape == x[0].shape and seen[-1][0] is x[0] and seen[-1][-1] is True
    y = delta_args()
    assert G.gated_delta_rule(*y).shape == y[2].shape and seen[-1][-2:] == (None, 1e-6)
    S.sample(torch.zeros((2, 5)), torch.zeros(2), top_k=3, temperature=torch.ones(2))
    assert seen[-1][6:] == (1.0, 3, 1.0, 0.0, False)
    ops = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            ops.append(str(func))
            return func(*args, **(kwargs or {}))
    with Watch():
        G.causal_conv(*x)
        G.gated_delta_rule(*y)
        S.sample(torch.zeros((2, 5)), torch.zeros(2))
    for name in ("causal_conv", "gated_delta_rule", "sample"):
        assert f"radiance.{name}.default" in ops


def test_fakes_have_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = lambda args: [mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args]  # noqa: E731
        assert G.causal_conv(*fake(conv_args())).shape == (3, 16)
        assert G.gated_delta_rule(*fake(delta_args())).shape == (3, 2, 64)
        logits, u = fake((torch.zeros((4, 9)), torch.zeros(4)))
        tokens, lp = S.sample(logits, u, logprobs=True)
        assert tokens.dtype == torch.int64 and tokens.shape == (4,) and lp.shape == (4,)
        assert S.sample(logits, u).shape == (4,)


@pytest.mark.parametrize("at", range(8))
def test_gradients_are_refused(seen, at):
    """These ops have none: an input that asks for one is an error and no silent cut."""
    args = list(delta_args())
    if not args[at].is_floating_point():
        return
    args[at] = args[at].clone().requires_grad_()
    try:
        out = G.gated_delta_rule(*args)
    except (RuntimeError, NotImplementedError):
        return
    if not out.requires_grad:
        pytest.fail("the gradient is cut without a word")
    with pytest.raises((RuntimeError, NotImplementedError)):
        out.sum().backward()
