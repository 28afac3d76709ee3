"""GPU parity of the attention over the 4-bit cache against the definition in float64 on the values
that the cache holds, within the bound that oracle.kv4_oracle.attention_tolerance derives."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, host_u16, to_dev
from tests._kv4 import Batch, bits
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def run(batch, max_q=None, max_len=None, **kw):
    q, cache, table, lens, starts, mq, ml = batch.device()
    print(f"[kv4] lens={batch.lens} q={batch.qs} heads={q.shape[1]}/{batch.Hkv} d={batch.d} "
          f"page={batch.page} {kw}", flush=True)
    out = K.attention(q, cache, table, lens, starts, max_q or mq, max_len or ml, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("Hq,Hkv,d,page,lens", [
    (1, 1, 64, 16, [1]), (4, 4, 64, 16, [33, 16, 1]), (32, 8, 128, 16, [500]),
    (7, 1, 128, 32, [1, 31, 32, 33, 127, 128, 129]), (16, 1, 128, 64, [700, 3]),
    (12, 4, 256, 32, [257, 100]), (32, 2, 64, 128, [1025, 6]), (17, 1, 64, 16, [300]),
    (40, 1, 128, 256, [900, 255, 256]), (70, 1, 128, 16, [77]), (34, 1, 256, 16, [140])])
def test_decode(Hq, Hkv, d, page, lens):
    b = Batch(np.random.default_rng(d + page), lens, [1] * len(lens), Hq, Hkv, d, page)
    b.check(run(b))


@pytest.mark.parametrize("Hq,Hkv,d,page,lens,qs", [
    (6, 2, 128, 16, [40, 100], [8, 3]), (4, 4, 64, 32, [17, 90, 5], [9, 2, 5]),
    (8, 1, 256, 64, [130, 7], [4, 7]), (48, 16, 128, 16, [200], [8]),
    (4, 1, 128, 16, [150, 64, 300], [150, 64, 20]), (14, 2, 128, 64, [333], [201]),
    (6, 1, 256, 16, [190, 80], [77, 80]), (8, 8, 64, 16, [260], [259]),
    (2, 1, 64, 128, [100, 1, 400], [100, 1, 1])])
@pytest.mark.parametrize("causal", [True, False])
def test_several_queries(Hq, Hkv, d, page, lens, qs, causal):
    b = Batch(np.random.default_rng(d + sum(qs)), lens, qs, Hq, Hkv, d, page)
    b.check(run(b, causal=causal), causal=causal)


@pytest.mark.parametrize("window", [1, 2, 15, 33, 100, 4096])
@pytest.mark.parametrize("d,lens,qs", [(128, [300, 40, 129], [1, 1, 1]), (64, [290, 33], [7, 33]),
                                       (256, [150, 200], [100, 3]), (128, [400], [220])])
def test_window(window, d, lens, qs):
    b = Batch(np.random.default_rng(window + d), lens, qs, 6, 2, d, 16)
    b.check(run(b, window=window), window=window)


@pytest.mark.parametrize("causal", [True, False])
def test_window_without_causal(causal):
    b = Batch(np.random.default_rng(3), [90, 200], [50, 2], 4, 2, 128, 32)
    b.check(run(b, causal=causal, window=40), causal=causal, window=40)


def test_long_context_is_split():
    """Chunks over workgroups, joined in a second launch; the same through a larger max_len, whose
    chunks are longer."""
    b = Batch(np.random.default_rng(4), [5000, 4097, 3, 129], [1, 2, 1, 2], 8, 2, 128, 64)
    assert _native_kv4.attention_workspace(6, 4, 2, 5000, 8, 2, 128, 0) > 0
    b.check(run(b))
    b.check(run(b, max_len=200000))
    b.check(run(b, max_q=9))


@pytest.mark.parametrize("n", [63, 64, 65, 150])
def test_many_sequences(n):
    """The runs are found 64 sequences at a time; most sequences empty, short ones, a long one at either
    end, and workgroups without work."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.choice([0, 0, 1, 17, 130, 300], n)]
    lens[0], lens[-1], lens[n // 2] = 700, 1000, 900
    qs = [int(x) for x in rng.choice([0, 1, 1, 2], n)]
    qs[0] = qs[-1] = qs[n // 2] = 1
    b = Batch(rng, lens, qs, 2, 1, 64, 16)
    b.check(run(b))
    b.check(run(b, window=40), window=40)


def test_batches_longer_than_they_are():
    """Limits far above the batch's lengths, as a graph's are: workgroups without work."""
    b = Batch(np.random.default_rng(21), [3, 900, 1], [1, 1, 1], 4, 2, 128, 16)
    b.check(run(b, max_len=1 << 20))
    b.check(run(b, max_q=4, max_len=1 << 20))
    b = Batch(np.random.default_rng(22), [1], [1], 4, 2, 256, 16)
    b.check(run(b, max_len=1 << 20))


def test_scores_far_apart_and_alike():
    """One key far above the others at either end; equal scores; large and tiny scales."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [700, 300], [2, 40], 4, 2, 128, 16, q_scale=12.0)
    b.check(run(b))
    b.check(run(b, scale=1e-4), scale=1e-4)
    b.check(run(b, scale=3.0), scale=3.0)
    b.q[:] = 0
    b.check(run(b))


def put(batch, seq, tok, head, what):
    """A NaN block in a token's key ('k') or value ('v')."""
    slot = batch.slots(seq)[tok]
    pk, pv, sk, sv = KO.places(int(slot % 16), batch.d)
    at = batch.cache[slot // batch.page, head, (slot % batch.page) // 16]
    at[(sk if what == "k" else sv)[tok % (batch.d // 32)]] = 255


@pytest.mark.parametrize("lens,qs,window", [([50, 200], [1, 1], 0), ([64, 190], [30, 190], 0),
                                            ([64, 190], [9, 170], 21), ([70], [70], 16)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_blocks_reach_those_who_see_them(lens, qs, window, d):
    """A NaN key makes its row NaN, a NaN value block its 32 channels, and only of queries that see
    the token: those before it (causal) and those past its window do not."""
    b = Batch(np.random.default_rng(6), lens, qs, 4, 2, d, 16)
    for s, n in enumerate(lens):
        put(b, s, n - 5, 0, "v")
        put(b, s, n // 2, 1, "v")
        put(b, s, n // 2 + 1, 1, "k")
        put(b, s, 3, 0, "k")
    b.check(run(b, window=window), window=window)


@pytest.mark.parametrize("fill", [0, 255])
def test_what_lies_behind_the_sequence_has_no_effect(fill):
    """The rest of the last page, and pages of nobody, hold NaN blocks and saturated codes."""
    b = Batch(np.random.default_rng(7), [37, 1, 15, 33, 190], [1, 1, 4, 33, 100], 4, 2, 128, 32)
    want = host_u16(run(b))
    used = np.zeros((b.pages, b.page), bool)
    for s in range(len(b.lens)):
        used.reshape(-1)[b.slots(s)] = True
    for p, t in np.argwhere(~used):
        for part in KO.places(int(t % 16), b.d):
            b.cache[p, :, t // 16, part] = fill
    assert np.array_equal(host_u16(run(b)), want)
    b.check(run(b))


def test_rows_that_see_nothing_are_zero():
    """More queries than cached tokens: the first ones stand before the sequence; empty sequences."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [5, 0, 20, 0], [9, 3, 1, 0], 4, 2, 128, 16)
    out = run(b)
    b.check(out)
    assert not out[:4].any() and not out[9:12].any() and out[4:9].any()
    b = Batch(rng, [3], [70], 2, 1, 64, 16)
    out = run(b)
    b.check(out)
    assert not out[:67].any() and out[67:].any()


def test_no_queries_and_no_sequences():
    b = Batch(np.random.default_rng(9), [20, 30], [0, 0], 4, 2, 128, 16)
    assert run(b, max_q=1).shape == (0, 4, 128)
    q, cache, table, _, _, _, _ = b.device()
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = K.attention(q, cache, table[:0], e, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 1)
    assert out.shape == (0, 4, 128)


def test_pages_outside_the_cache_make_their_queries_nan():
    b = Batch(np.random.default_rng(10), [100, 100, 100, 100], [1, 1, 2, 1], 4, 2, 128, 16)
    b.table[0, 3], b.table[2, 6] = b.pages, -1
    out = O.bf16_to_f32(host_u16(run(b)))
    assert np.isnan(out[0]).all() and np.isnan(out[2:4]).all()
    b.check(run(b), only=(1, 3))


def test_sequences_past_the_limits_are_nan():
    """A length past max_len or the table's row, more queries than max_q: the kernels see what the host
    does not, and the other sequences are right."""
    b = Batch(np.random.default_rng(11), [60, 100, 50, 20], [2, 1, 1, 2], 4, 2, 128, 16)
    q, cache, table, lens, starts, mq, ml = b.device()
    out = O.bf16_to_f32(host_u16(K.attention(q, cache, table, lens, starts, 2, 60)))
    assert np.isnan(out[2]).all() and not np.isnan(np.delete(out, 2, 0)).any()
    out = O.bf16_to_f32(host_u16(K.attention(q, cache, table, lens, starts, 1, 100)))
    assert np.isnan(out[[0, 1, 4, 5]]).all() and not np.isnan(out[2:4]).any()
    lens[1] = 2000
    out = O.bf16_to_f32(host_u16(K.attention(q, cache, table, lens, starts, 2, 4000)))
    assert np.isnan(out[2]).all() and not np.isnan(np.delete(out, 2, 0)).any()
    b.check(run(b))


def test_strides_of_queries_tables_and_pages():
    """Queries inside wider heads and off 16 bytes, a table inside a larger one, layers side by side."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [70, 33], [3, 1], 4, 2, 128, 32)
    want = host_u16(run(b))
    q, cache, table, lens, starts, mq, ml = b.device()
    wide = torch.zeros((4, 4, 256), dtype=torch.bfloat16, device="cuda")
    wide[..., 128:] = q
    odd = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = q.reshape(-1)
    big = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    big[:, 5:5 + table.shape[1]] = table
    layers = torch.zeros((cache.shape[0], 3, *cache.shape[1:]), dtype=torch.uint8, device="cuda")
    layers[:, 2] = cache
    for args in ((wide[..., 128:], cache, table), (odd[1:].view(q.shape), cache, table),
                 (q, cache, big[:, 5:]), (q, layers[:, 2], table),
                 (q, cache, table.T.contiguous().T)):
        out = K.attention(*args, lens, starts, mq, ml)
        assert np.array_equal(host_u16(out), want)


def test_offsets_past_32_bits():
    """Pages more than 2^32 bytes into the cache."""
    b = Batch(np.random.default_rng(13), [200, 90], [1, 40], 8, 2, 128, 64)
    page = b.cache[0].nbytes
    far = (1 << 32) // page + 1000
    q, cache, table, lens, starts, mq, ml = b.device()
    big = torch.empty((far + b.pages, *cache.shape[1:]), dtype=torch.uint8, device="cuda")
    assert big.numel() > 1 << 32
    big[far:] = cache
    out = K.attention(q, big, torch.where(table >= 0, table + far, table), lens, starts, mq, ml)
    b.check(out)
    slots = b.slots(0)[:20]
    k, v = K.gather(big, to_dev(slots + far * b.page))
    wk, wv = KO.read(b.cache, slots)
    assert np.array_equal(O.bf16_to_f32(host_u16(k)), wk.astype(np.float32))
    assert np.array_equal(O.bf16_to_f32(host_u16(v)), wv.astype(np.float32))


def test_same_bits_every_time():
    b = Batch(np.random.default_rng(14), [4000, 900], [1, 70], 8, 2, 128, 16)
    first = host_u16(run(b))
    for _ in range(3):
        assert np.array_equal(host_u16(run(b)), first)


def test_graph_of_a_batch_serves_other_lengths():
    """Captured with the limits of the batch: the lengths, pages and queries are read on replay."""
    rng = np.random.default_rng(15)
    b = Batch(rng, [900, 300, 40], [1, 1, 1], 8, 2, 128, 16)
    q, cache, table, lens, starts, _, _ = b.device()
    K.attention(q, cache, table, lens, starts, 1, 1000)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = K.attention(q, cache, table, lens, starts, 1, 1000)
    for lens_now in ([900, 300, 40], [1, 250, 40], [850, 0, 17]):
        b.lens = lens_now
        lens.copy_(torch.tensor(lens_now, dtype=torch.int32))
        b.q = bits(rng, 3, 8, 128, scale=1.5)
        q.copy_(bf16_dev(b.q))
        g.replay()
        torch.cuda.synchronize()
        b.check(out)
        eager = K.attention(q, cache, table, lens, starts, 1, 1000)
        assert torch.equal(eager, out)


def test_other_streams():
    """Called on a stream that is not the tensors' own, behind an event; the workspace is that
    stream's."""
    b = Batch(np.random.default_rng(16), [3000, 2000], [1, 1], 8, 2, 128, 16)
    want = host_u16(run(b))
    q, cache, table, lens, starts, mq, ml = b.device()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        for _ in range(4):
            outs.append(K.attention(q, cache, table, lens, starts, mq, ml))
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert np.array_equal(host_u16(o), want)


def test_op_is_one_opaque_node_under_compile():
    b = Batch(np.random.default_rng(17), [60], [1], 4, 2, 128, 16)
    args = b.device()
    fn = torch.compile(lambda q, c, t, n, s: K.attention(q, c, t, n, s, 1, 60) * 2, backend="eager",
                       fullgraph=True)
    assert torch.equal(fn(*args[:5]), K.attention(*args[:5], 1, 60) * 2)
