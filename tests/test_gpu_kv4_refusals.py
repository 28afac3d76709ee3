"""What the ops of the 4-bit cache refuse before a launch, with which words; and that the call after a
refusal is served."""
import pytest
import torch

from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def bf(*shape):
    return torch.ones(shape, dtype=torch.bfloat16, device="cuda")


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def rope(**kw):
    a = dict(q=bf(3, 4, 128), k=bf(3, 2, 128), q_weight=bf(128), k_weight=bf(128),
             cos_sin=torch.ones((9, 64), device="cuda"), positions=ints(0, 1, 2, dtype=torch.int64))
    a.update(kw)
    return K.qk_norm_rope(**a)


def append(**kw):
    a = dict(q=bf(3, 4, 128), k=bf(3, 2, 128), v=bf(3, 2, 128), q_weight=None, k_weight=None,
             cos_sin=None, positions=None, cache=K.new_cache(4, 2, 16, 128),
             slots=ints(0, 1, 2, dtype=torch.int64))
    a.update(kw)
    return K.qk_norm_rope_append(**a)


def attention(**kw):
    a = dict(q=bf(3, 4, 128), cache=K.new_cache(4, 2, 16, 128), page_table=torch.zeros(
        (2, 2), dtype=torch.int32, device="cuda"), seq_lens=ints(5, 6), q_starts=ints(0, 1, 3),
             max_q=2, max_len=6)
    a.update(kw)
    return K.attention(**a)


def move(cache=None, pairs=((0, 1),), table=None, host=True):
    cache = K.new_cache(4, 2, 16, 128, layers=2) if cache is None else cache
    pairs = torch.tensor(pairs, dtype=torch.int32)
    return K.move_pages(cache, pairs if host else pairs.cuda(), table)


REFUSED = [
    (rope, dict(q=lambda: bf(3, 4)), "", "q must be bf16"),
    (rope, dict(q=lambda: bf(3, 4, 128).float()), "", "q must be bf16"),
    (rope, dict(q=lambda: bf(3, 4, 96), k=lambda: bf(3, 2, 96)), "", "head size 96"),
    (rope, dict(k=lambda: bf(2, 2, 128)), "", "k BFloat16 .2, 2, 128. does not match"),
    (rope, dict(k=lambda: bf(3, 2, 64)), "", "does not match"),
    (rope, dict(q_weight=lambda: bf(64)), "", "q_weight must be bf16 .128."),
    (rope, dict(k_weight=lambda: bf(128).float()), "", "k_weight must be bf16"),
    (rope, dict(cos_sin=lambda: torch.ones((9, 64), device="cuda").half()), "", "cos_sin must be"),
    (rope, dict(cos_sin=lambda: torch.ones((9, 24), device="cuda")), "", "24 rotated channels"),
    (rope, dict(cos_sin=lambda: torch.ones((9, 144), device="cuda")), "", "144 rotated channels"),
    (rope, dict(positions=lambda: None), "", "positions must be"),
    (rope, dict(positions=lambda: ints(0, 1)), "", "positions must be"),
    (rope, dict(positions=lambda: bf(3)), "", "positions must be"),
    (rope, dict(positions=lambda: torch.zeros((0, 3), dtype=torch.int64, device="cuda")), "", "positions"),
    (rope, dict(positions=lambda: torch.zeros((2, 3), dtype=torch.int64, device="cuda")), "", "2 axes need"),
    (rope, dict(axis=lambda: ints(0, 0)), "", "axis must be int32 .32."),
    (rope, dict(k=lambda: bf(3, 2, 128).cpu()), "", "tensors on cuda:0 and cpu"),
    (append, dict(v=lambda: bf(3, 4, 128)), "", "v BFloat16"),
    (append, dict(slots=lambda: ints(0, 1, 2)), "", "slots must be int64 .3."),
    (append, dict(slots=lambda: ints(0, 1, dtype=torch.int64)), "", "slots must be int64"),
    (append, dict(cache=lambda: K.new_cache(4, 2, 16, 64)), "", "cache of head size 64"),
    (append, dict(cache=lambda: K.new_cache(4, 3, 16, 128)), "", "cache of 3 kv heads"),
    (append, dict(cache=lambda: K.new_cache(4, 2, 16, 128, layers=1)), "", "one layer's"),
    (append, dict(cache=lambda: K.new_cache(4, 2, 32, 128)[:, :, :1]), "", "contiguous and 16-byte"),
    (append, dict(cache=lambda: K.new_cache(4, 2, 16, 128).view(torch.int8)), "", "cache must be uint8"),
    (attention, dict(q=lambda: bf(3, 3, 128)), "", "3 query heads over 2"),
    (attention, dict(q=lambda: bf(3, 4, 64)), "", "cache of head size 128"),
    (attention, dict(seq_lens=lambda: ints(5, 6, dtype=torch.int64)), "", "seq_lens must be int32"),
    (attention, dict(q_starts=lambda: ints(0, 3)), "", "q_starts must be int32 .3."),
    (attention, dict(page_table=lambda: ints(0, 1)), "", "page_table must be int32"),
    (attention, dict(page_table=lambda: torch.zeros((3, 2), dtype=torch.int32, device="cuda")), "", "page_table"),
    (attention, dict(), dict(max_q=-1), "max_q=-1"), (attention, dict(), dict(max_len=2 ** 31 - 1), "max_len"),
    (attention, dict(), dict(max_q=2 ** 31), "max_q=2147483648 is out of range"),
    (attention, dict(), dict(window=-2), "window=-2"), (attention, dict(), dict(scale=0.0), "scale"),
    (attention, dict(), dict(scale=float("nan")), "scale"),
    (move, dict(), dict(pairs=((0, 4),)), "outside"), (move, dict(), dict(pairs=((0, 1), (1, 2))), "both"),
    (move, dict(), dict(pairs=((0, 2), (1, 2))), "twice"), (move, dict(), dict(host=False), "on the host"),
    (move, dict(), dict(pairs=((0, 1, 2),)), "pairs must be"),
    (move, dict(table=lambda: bf(2, 2)), "", "page_table must be"),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused(i):
    call, tensors, values, words = REFUSED[i]
    with pytest.raises(RuntimeError, match=words) as e:
        call(**{k: f() for k, f in tensors.items()}, **(values or {}))
    assert str(e.value).startswith("[radiance.kv4] ")


def test_served_after_refusals():
    q, k = rope()
    assert q.shape == (3, 4, 128) and append().shape == (3, 4, 128) and attention().shape == (3, 4, 128)
    move()
    torch.cuda.synchronize()


def test_gradients_are_refused():
    q = bf(3, 4, 128).requires_grad_()
    with pytest.raises(RuntimeError):
        attention(q=q).sum().backward()
