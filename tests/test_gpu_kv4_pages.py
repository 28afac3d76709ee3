"""Page moves of the 4-bit cache on the GPU: bytes and page numbers, exactly."""
import numpy as np
import pytest
import torch

from tests._check import host_u8, to_dev
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def moved(cache, pairs, table):
    """cache [layers, pages, ...] and table after the moves, on the host."""
    c, t = cache.copy(), None if table is None else table.copy()
    for a, b in pairs:
        c[:, b] = cache[:, a]
        if t is not None:
            t[table == a] = b
    return c, t


@pytest.mark.parametrize("layers,pages,H,page,d,n,rows,cols", [
    (1, 2, 1, 16, 64, 1, 1, 1), (3, 40, 2, 16, 128, 16, 3, 50), (2, 60, 3, 32, 64, 17, 1, 257),
    (5, 1100, 1, 16, 64, 500, 7, 300), (2, 9, 16, 256, 128, 4, 2, 3), (1, 2000, 1, 16, 64, 900, 40, 11)])
def test_moves(layers, pages, H, page, d, n, rows, cols):
    rng = np.random.default_rng(n)
    cache = rng.integers(0, 256, (layers, pages, H, page // 16, 17 * d), dtype=np.uint8)
    pairs = rng.permutation(pages)[:2 * n].reshape(n, 2).astype(np.int32)
    table = rng.integers(-1, pages, (rows, cols)).astype(np.int32)
    c, t = to_dev(cache), to_dev(table)
    K.move_pages(c, torch.from_numpy(pairs), t)
    wc, wt = moved(cache, pairs, table)
    assert np.array_equal(host_u8(c), wc) and np.array_equal(t.cpu().numpy(), wt)
    one = to_dev(cache[0])                              # a layer alone, no table
    K.move_pages(one, torch.from_numpy(pairs))
    assert np.array_equal(host_u8(one), wc[0])


def test_one_page_to_several_and_strided_caches():
    """A fork copies a page more than once; layers inside pages, a table inside a larger one."""
    rng = np.random.default_rng(1)
    cache = rng.integers(0, 256, (3, 12, 2, 1, 17 * 64), dtype=np.uint8)
    pairs = np.array([[4, 1], [4, 9], [5, 2]], np.int32)
    whole = to_dev(np.ascontiguousarray(cache.transpose(1, 0, 2, 3, 4)))      # [pages, layers, ...]
    K.move_pages(whole.transpose(0, 1), torch.from_numpy(pairs))
    assert np.array_equal(host_u8(whole.transpose(0, 1).contiguous()), moved(cache, pairs, None)[0])
    big = rng.integers(0, 12, (4, 30)).astype(np.int32)
    t = to_dev(big)
    K.move_pages(to_dev(cache), torch.tensor([[3, 7]], dtype=torch.int32), t[:, 4:11])
    want = big.copy()
    want[:, 4:11][big[:, 4:11] == 3] = 7
    assert np.array_equal(t.cpu().numpy(), want)


def test_nothing_to_move():
    cache = K.new_cache(4, 2, 16, 64)
    t = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    K.move_pages(cache, torch.zeros((0, 2), dtype=torch.int32), t)
    K.move_pages(cache, torch.tensor([[0, 1]], dtype=torch.int32), t[:, :0])
    assert t.tolist() == [[0, 1, 2, 3]]


def test_moves_past_32_bits():
    page = 2 * 17 * 64
    far = (1 << 32) // page + 5
    cache = torch.empty((far + 2, 2, 1, 17 * 64), dtype=torch.uint8, device="cuda")
    x = torch.randint(0, 256, cache[0].shape, dtype=torch.uint8, device="cuda")
    cache[1] = x
    K.move_pages(cache, torch.tensor([[1, far]], dtype=torch.int32))
    assert torch.equal(cache[far], x)
    cache[2] = 0
    K.move_pages(cache, torch.tensor([[far, 2]], dtype=torch.int32))
    assert torch.equal(cache[2], x)


def test_graph_of_a_move():
    """The pairs are the launch's own: the graph needs no list kept alive."""
    cache = K.new_cache(6, 1, 16, 64)
    K.move_pages(cache, torch.tensor([[0, 1]], dtype=torch.int32))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.move_pages(cache, torch.tensor([[2, 3], [2, 5]], dtype=torch.int32))
    for i in range(3):
        cache[2] = i + 7
        g.replay()
        torch.cuda.synchronize()
        assert (cache[3] == i + 7).all() and (cache[5] == i + 7).all() and not cache[4].any()
