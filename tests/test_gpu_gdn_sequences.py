"""The sequences of the example's stack where they have no tokens, none yet, or more than there is room for."""
import numpy as np
import pytest
import torch

from examples.gdn_generate import DRAFT, Hybrid
from tests.test_gpu_gdn_generate import close
from vllm_sly_radiance_amd import _native, _native_decode, _native_kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native.lib(), _native_kv4.lib(), _native_decode.lib()


@torch.no_grad()
def test_a_fork_of_nothing_begins_from_nothing():
    s = Hybrid(layers=4, pages=96)
    rng = np.random.default_rng(5)
    tokens = rng.integers(0, 512, 50).tolist()
    a = s.add()
    s.forward([a], [tokens[:4]], drafts=True)           # states that are not zero in the last slots
    b = s.add()
    c = s.fork(b)
    want = s.forward([b], [tokens])[-1]
    close(s.forward([c], [tokens])[-1], want)


@torch.no_grad()
def test_a_sequence_without_tokens_among_drafts_keeps_its_state():
    s = Hybrid(layers=4, pages=96)
    rng = np.random.default_rng(6)
    tokens = rng.integers(0, 512, 50).tolist()
    a, b, c = s.add(), s.add(), s.add()
    s.forward([a, b, c], [tokens, tokens, tokens[::-1]])
    want = s.forward([a], [tokens[:1]])[-1]
    s.forward([b, c], [[], tokens[:2]], drafts=True)
    close(s.forward([b], [tokens[:1]])[-1], want)


@torch.no_grad()
def test_more_drafts_than_a_sequence_has_slots_are_refused():
    s = Hybrid(layers=4, pages=96)
    a = s.add()
    s.forward([a], [[1, 2, 3]])
    before = s.conv_state.clone(), s.state.clone(), dict(s.now), s.pool.length(a)
    with pytest.raises(ValueError, match="drafted"):
        s.forward([a], [list(range(2 + DRAFT))], drafts=True)
    assert torch.equal(before[0], s.conv_state) and torch.equal(before[1], s.state)
    assert before[2:] == (s.now, s.pool.length(a))


def test_no_room_for_a_sequence_changes_nothing():
    s = Hybrid(layers=1, pages=96, sequences=1)
    a = s.add()
    for more in (s.add, lambda: s.fork(a)):
        with pytest.raises(RuntimeError, match="1 sequences, as many as"):
            more()
    s.drop(a)
    assert not s.pool._sequences and s.free == [0]
