"""GPU parity of the attention over the 4-bit cache where a call has many query rows (prompt chunks,
alone and beside decoding sequences) against the definition in float64 on the values that the cache
holds, within the bound that oracle.kv4_oracle.attention_tolerance derives."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import host_u16, to_dev
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def run(batch, max_q=None, max_len=None, **kw):
    q, cache, table, lens, starts, mq, ml = batch.device()
    # rows enough for workgroups of many rows (tests/test_kv4_abi_cpu.py has the rule)
    assert q.shape[0] * q.shape[1] >= 200 * (32 if batch.d == 256 else 64)
    print(f"[kv4] lens={batch.lens} q={batch.qs} heads={q.shape[1]}/{batch.Hkv} d={batch.d} "
          f"page={batch.page} {kw}", flush=True)
    out = K.attention(q, cache, table, lens, starts, max_q or mq, max_len or ml, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("Hq,Hkv,d,page,lens,qs", [
    (64, 64, 64, 16, [300, 257, 400], [290, 257, 160]),     # every head its own keys
    (64, 8, 64, 64, [900], [701]),
    (64, 8, 128, 32, [700], [700]),
    (48, 16, 128, 16, [513, 129, 640], [500, 129, 310]),
    (32, 1, 128, 256, [64, 130, 1300], [64, 130, 1210]),
    (24, 4, 256, 32, [500, 33, 470], [470, 32, 450]),
    (16, 2, 256, 128, [1410], [1401]),
])
def test_chunks(Hq, Hkv, d, page, lens, qs):
    b = Batch(np.random.default_rng(1), lens, qs, Hq, Hkv, d, page)
    b.check(run(b))


@pytest.mark.parametrize("d,Hq,Hkv,qs", [(128, 64, 8, [1, 300, 1, 2, 290, 0, 3, 130]),
                                         (64, 96, 4, [200, 1, 270, 1]),
                                         (256, 32, 4, [1, 1, 1, 700, 3, 4]),
                                         (128, 128, 1, [1, 200, 160])])
def test_chunks_beside_decoding_sequences(d, Hq, Hkv, qs):
    """Sequences of few rows, which attn_rows serves, and of none among prompt chunks; rows that see
    nothing and rows whose sequence is longer than the chunk."""
    rng = np.random.default_rng(2)
    lens = [max(0, n + int(rng.integers(-3, 400))) if n != 300 else 290 for n in qs]
    b = Batch(rng, lens, qs, Hq, Hkv, d, 16)
    out = run(b)
    b.check(out)
    if 300 in qs:
        at = int(b.starts[qs.index(300)])
        assert not out[at:at + 10].any() and out[at + 10].any()


@pytest.mark.parametrize("d,Hq,Hkv,qs", [(64, 32, 8, [350, 8, 7, 9, 8, 16, 17, 1]),
                                         (128, 32, 8, [8, 9, 7, 350, 8, 16, 17, 0]),
                                         (128, 32, 4, [5, 400, 4, 1, 2, 4, 5, 3]),
                                         (256, 24, 4, [4, 300, 5, 6, 3, 4])])
def test_chunk_beside_drafts(d, Hq, Hkv, qs):
    """Sequences of a few queries each beside a chunk: up to what the others have on average, and beyond."""
    rng = np.random.default_rng(50)
    lens = [n + int(rng.integers(0, 500)) for n in qs]
    b = Batch(rng, lens, qs, Hq, Hkv, d, 16)
    b.check(run(b))
    b.check(run(b, window=150), window=150)


def test_more_sequences_than_lanes():
    """The tiles of a batch are found 64 sequences at a time."""
    rng = np.random.default_rng(3)
    qs = [(20, 1, 0, 13)[i % 4] for i in range(150)]
    b = Batch(rng, [n + int(rng.integers(0, 60)) for n in qs], qs, 64, 2, 64, 16)
    b.check(run(b))


PARTS = [(16, 2, 64, 16, [1500], [800]), (8, 2, 256, 64, [1400], [801]), (32, 2, 128, 32, [1100], [401]),
         (32, 2, 128, 32, [1100, 1000], [399, 399]),        # every sequence alike but for its length
         (32, 2, 128, 16, [1300, 900, 20], [300, 290, 1])]


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 333)])
@pytest.mark.parametrize("i", range(len(PARTS)))
def test_units_in_parts(i, causal, window):
    """Few units over long contexts: their tokens are cut into parts, some of which a row sees none of."""
    Hq, Hkv, d, page, lens, qs = PARTS[i]
    b = Batch(np.random.default_rng(20 + i), lens, qs, Hq, Hkv, d, page)
    # (a window leaves some of them too few tokens to be cut)
    assert _native_kv4.attention_workspace(sum(qs), len(qs), max(qs), max(lens), Hq, Hkv, d, 0) > 4096
    b.check(run(b, causal=causal, window=window), causal=causal, window=window)


def test_parts_with_nan_blocks_bad_pages_and_bad_lengths():
    b = Batch(np.random.default_rng(30), [1200, 1100, 1150], [300, 300, 300], 16, 2, 128, 16)
    for s, tok, head, what in ((0, 100, 0, "v"), (0, 700, 1, "k"), (0, 1150, 1, "v"), (2, 1149, 0, "v")):
        slot = b.slots(s)[tok]
        pk, pv, sk, sv = KO.places(int(slot % 16), 128)
        b.cache[slot // 16, head, 0][(sk if what == "k" else sv)[tok % 4]] = 255
    b.check(run(b))
    page = b.table[1, 60]
    b.table[1, 60] = -1
    out = run(b)
    got = O.bf16_to_f32(host_u16(out))
    # rows of the second sequence that come after token 960, and those of their workgroup
    assert np.isnan(got[300 + 160:600]).all()
    b.check(out, only=(0, 2))
    b.table[1, 60] = page
    q, cache, table, lens, starts, mq, ml = b.device()
    for bad in (0, 1, 2):
        wrong = lens.clone()
        wrong[bad] = 5000
        got = O.bf16_to_f32(host_u16(K.attention(q, cache, table, wrong, starts, mq, ml)))
        assert np.isnan(got[300 * bad:300 * bad + 300]).all()
        b.check(K.attention(q, cache, table, wrong, starts, mq, ml), only={0, 1, 2} - {bad})


@pytest.mark.parametrize("window", [1, 31, 64, 200, 5000])
@pytest.mark.parametrize("causal", [True, False])
def test_window(window, causal):
    b = Batch(np.random.default_rng(4), [600, 150, 90], [220, 140, 1], 128, 16, 128, 32)
    b.check(run(b, window=window, causal=causal), window=window, causal=causal)


def test_not_causal_wide():
    b = Batch(np.random.default_rng(5), [300, 400], [250, 200], 64, 8, 256, 64)
    b.check(run(b, causal=False), causal=False)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("window", [0, 75])
def test_nan_blocks_reach_those_who_see_them(d, page, window):
    """NaN keys and NaN value blocks, in the first tokens, in later steps and several in one step, and
    only of queries that see them."""
    b = Batch(np.random.default_rng(6), [390, 360, 5], [360, 355, 1], 64, 4, d, page)
    for s, tok, head, what in ((0, 0, 0, "v"), (0, 200, 1, "v"), (0, 201, 1, "v"), (0, 333, 2, "k"),
                               (1, 130, 3, "v"), (1, 359, 0, "v"), (1, 64, 1, "k"), (2, 3, 2, "v")):
        slot = b.slots(s)[tok]
        pk, pv, sk, sv = KO.places(int(slot % 16), d)
        at = b.cache[slot // page, head, (slot % page) // 16]
        at[(sk if what == "k" else sv)[tok % (d // 32)]] = 255
    b.check(run(b, window=window), window=window)


def test_scores_far_apart_and_alike():
    rng = np.random.default_rng(7)
    b = Batch(rng, [720, 20], [700, 1], 64, 8, 128, 16, q_scale=12.0)
    b.check(run(b))
    b.check(run(b, scale=1e-4), scale=1e-4)
    b.q[:] = 0
    b.check(run(b))


@pytest.mark.parametrize("fill", [0, 255])
def test_what_lies_behind_the_sequence_has_no_effect(fill):
    b = Batch(np.random.default_rng(8), [417, 333, 30], [400, 320, 1], 64, 4, 128, 64)
    want = host_u16(run(b))
    used = np.zeros((b.pages, b.page), bool)
    for s in range(len(b.lens)):
        used.reshape(-1)[b.slots(s)] = True
    for p, t in np.argwhere(~used):
        for part in KO.places(int(t % 16), b.d):
            b.cache[p, :, t // 16, part] = fill
    assert np.array_equal(host_u16(run(b)), want)


def test_pages_outside_the_cache_and_bad_lengths_are_nan():
    """A page outside the cache makes a chunk's rows that read it NaN; a sequence past max_len is NaN;
    the others are right."""
    b = Batch(np.random.default_rng(9), [300, 300, 300, 40], [250, 250, 250, 1], 64, 8, 128, 16)
    b.table[1, 17] = b.pages + 5
    out = run(b)
    got = O.bf16_to_f32(host_u16(out))
    assert np.isnan(got[499]).all()
    b.check(out, only=(0, 2, 3))
    q, cache, table, lens, starts, mq, ml = b.device()
    lens[2] = 4000
    got = O.bf16_to_f32(host_u16(K.attention(q, cache, table, lens, starts, mq, ml)))
    assert np.isnan(got[500:750]).all() and not np.isnan(got[:250]).any() and not np.isnan(got[750]).any()


def test_strides_and_far_pages():
    """Queries inside wider heads, a table inside a larger one, layers side by side, and pages more than
    2^32 bytes into the cache."""
    b = Batch(np.random.default_rng(10), [500, 250], [470, 235], 64, 8, 128, 32)
    want = host_u16(run(b))
    q, cache, table, lens, starts, mq, ml = b.device()
    wide = torch.zeros((q.shape[0], 64, 192), dtype=torch.bfloat16, device="cuda")
    wide[..., 64:] = q
    big = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    big[:, 5:5 + table.shape[1]] = table
    layers = torch.zeros((cache.shape[0], 3, *cache.shape[1:]), dtype=torch.uint8, device="cuda")
    layers[:, 1] = cache
    far = (1 << 32) // b.cache[0].nbytes + 100
    huge = torch.empty((far + b.pages, *cache.shape[1:]), dtype=torch.uint8, device="cuda")
    huge[far:] = cache
    for args in ((wide[..., 64:], cache, table), (q, cache, big[:, 5:]), (q, layers[:, 1], table),
                 (q, huge, torch.where(table >= 0, table + far, table))):
        assert np.array_equal(host_u16(K.attention(*args, lens, starts, mq, ml)), want)
    b.check(run(b))


def test_graph_of_a_batch_serves_other_lengths():
    """A captured call answers for the lengths and starts of each replay."""
    rng = np.random.default_rng(11)
    qs = [[400, 1, 310], [150, 2, 559], [711, 0, 0]]
    b = [Batch(rng, [n + 60 for n in x], x, 64, 8, 128, 16) for x in qs]
    cols = max(x.table.shape[1] for x in b)
    pages = max(x.pages for x in b)
    q = torch.zeros((711, 64, 128), dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((pages, *b[0].cache.shape[1:]), dtype=torch.uint8, device="cuda")
    table = torch.zeros((3, cols), dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")

    def load(x):
        dq, dc, dt, dl, ds, _, _ = x.device()
        q.zero_()
        q[:dq.shape[0]] = dq[:711]
        cache[:dc.shape[0]] = dc
        table[:, :dt.shape[1]] = dt
        lens.copy_(dl)
        starts.copy_(ds)
        torch.cuda.synchronize()

    load(b[0])
    K.attention(q, cache, table, lens, starts, 711, 800)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            out = K.attention(q, cache, table, lens, starts, 711, 800)
    for x in (b[1], b[0], b[2], b[1]):
        load(x)
        g.replay()
        torch.cuda.synchronize()
        x.check(out[:sum(x.qs)])
        assert torch.equal(out, K.attention(q, cache, table, lens, starts, 711, 800))


def test_same_bits_every_time_and_on_another_stream():
    b = Batch(np.random.default_rng(12), [900, 300], [620, 90], 64, 8, 128, 16)
    args = b.device()
    want = host_u16(K.attention(*args))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [K.attention(*args) for _ in range(3)]
    s.synchronize()
    for out in outs:
        assert np.array_equal(host_u16(out), want)


def test_one_chunk_among_many_decoding_and_bad_sequences():
    """Far fewer row tiles than the longest chunk's times the batch, and bad sequences among them."""
    rng = np.random.default_rng(40)
    qs = [1] * 70
    qs[33] = 600
    lens = [int(n) for n in rng.integers(1, 90, 70)]
    lens[33] = 650
    b = Batch(rng, lens, qs, 32, 2, 64, 16)
    b.check(run(b))
    q, cache, table, dl, starts, mq, ml = b.device()
    bad = (0, 7, 32, 34, 69)
    for i in bad:
        dl[i] = ml + 1 + i
    out = K.attention(q, cache, table, dl, starts, mq, ml)
    got = O.bf16_to_f32(host_u16(out))
    for i in bad:
        assert np.isnan(got[b.starts[i]:b.starts[i + 1]]).all()
    b.check(out, only=set(range(70)) - set(bad))
