"""GPU parity of the head norm + rotation and of the append to the 4-bit cache: every step is fixed, so
the bf16 outputs and the cache's bytes are the oracle's bits; and the definition in float64."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, host_u16, host_u8, to_dev
from tests._kv4 import angles, bits
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu
ROWS = 300


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def same_bits(got, want, what):
    """bf16 bits equal, any NaN for a NaN."""
    nan = np.isnan(O.bf16_to_f32(want))
    assert np.array_equal(np.isnan(O.bf16_to_f32(got)), nan), f"{what}: NaN places differ"
    bad = np.argwhere((got != want) & ~nan)
    assert bad.size == 0, f"{what}: {len(bad)} differ, first at {bad[:3].tolist()}"


def case(seed, T, Hq, Hkv, d, rot, axes=1):
    rng = np.random.default_rng(seed)
    qkv = bits(rng, T, (Hq + 2 * Hkv) * d, scale=2.0)
    qw, kw = bits(rng, d, scale=0.2), bits(rng, d, scale=0.2, mean=1.0)
    table = angles(ROWS, rot) if rot else None
    pos = rng.integers(0, ROWS, (axes, T))
    axis = rng.integers(0, axes, rot // 2).astype(np.int32) if axes > 1 else None
    x = bf16_dev(qkv)
    dev = [x[:, :Hq * d].unflatten(1, (Hq, d)), x[:, Hq * d:(Hq + Hkv) * d].unflatten(1, (Hkv, d)),
           x[:, (Hq + Hkv) * d:].unflatten(1, (Hkv, d))]
    host = [qkv[:, :Hq * d].reshape(T, Hq, d), qkv[:, Hq * d:(Hq + Hkv) * d].reshape(T, Hkv, d),
            qkv[:, (Hq + Hkv) * d:].reshape(T, Hkv, d)]
    return rng, host, dev, qw, kw, table, pos, axis


def dev_pos(pos, dtype=np.int64):
    p = to_dev(pos.astype(dtype))
    return p[0] if pos.shape[0] == 1 else p


@pytest.mark.parametrize("T,Hq,Hkv,d,rot,axes,adjacent,plus_one", [
    (1, 32, 8, 128, 128, 1, False, True), (1, 1, 1, 64, 64, 1, False, False),
    (3, 4, 4, 64, 32, 2, False, True), (9, 6, 2, 64, 64, 3, True, False),
    (5, 3, 1, 128, 16, 1, False, False), (7, 4, 2, 128, 96, 3, False, True),
    (130, 5, 1, 128, 128, 4, True, True), (2, 8, 2, 256, 64, 3, False, True),
    (67, 24, 4, 256, 256, 1, False, False), (33, 2, 2, 256, 32, 1, True, True),
    (700, 16, 8, 128, 128, 1, False, False), (8, 2, 1, 128, 0, 1, False, True)])
def test_rope_bits(T, Hq, Hkv, d, rot, axes, adjacent, plus_one):
    _, host, dev, qw, kw, table, pos, axis = case(T + d, T, Hq, Hkv, d, rot, axes)
    q, k = K.qk_norm_rope(dev[0], dev[1], bf16_dev(qw), bf16_dev(kw),
                          None if table is None else to_dev(table), dev_pos(pos),
                          axis=None if axis is None else to_dev(axis), eps=1e-6, plus_one=plus_one,
                          adjacent=adjacent)
    for got, x, w, name in ((q, host[0], qw, "q"), (k, host[1], kw, "k")):
        args = (x, w, table, pos, axis, 1e-6, plus_one, adjacent)
        assert got.is_contiguous() and tuple(got.shape) == x.shape
        same_bits(host_u16(got), O.f32_to_bf16(KO.norm_rope(*args)), name)
        exact = KO.norm_rope(*args, dtype=np.float64)
        # one rounding to bf16, and the fp32 steps against the pair's magnitudes
        near = np.abs(KO.norm_rope(x, w, None, None, plus_one=plus_one, dtype=np.float64)).max(-1)
        off = np.abs(O.bf16_to_f32(host_u16(got)).astype(np.float64) - exact)
        assert (off <= 2.0 ** -8 * np.abs(exact) + 2.0 ** -18 * near[..., None]).all()


@pytest.mark.parametrize("table_type,pos_type", [("bf16", np.int32), ("fp32", np.int32),
                                                 ("bf16", np.int64)])
def test_rope_table_and_position_types(table_type, pos_type):
    _, host, dev, qw, kw, table, pos, axis = case(5, 21, 4, 2, 128, 64, 2)
    t = to_dev(table)
    if table_type == "bf16":
        t = t.to(torch.bfloat16)
        table = O.bf16_to_f32(host_u16(t))
    q, k = K.qk_norm_rope(dev[0], dev[1], bf16_dev(qw), bf16_dev(kw), t, dev_pos(pos, pos_type),
                          axis=to_dev(axis))
    same_bits(host_u16(q), O.f32_to_bf16(KO.norm_rope(host[0], qw, table, pos, axis)), "q")
    same_bits(host_u16(k), O.f32_to_bf16(KO.norm_rope(host[1], kw, table, pos, axis)), "k")


def test_rope_layouts():
    """Heads inside wider heads, transposed heads, off 16 bytes, broadcast tokens, strided positions
    and weights; one tensor's norm left out."""
    rng, _, _, qw, kw, table, pos, _ = case(8, 10, 4, 2, 128, 128)
    wide = bits(rng, 10, 4, 256)                        # queries beside their gates
    kt = bits(rng, 2, 10, 128)                          # [heads, tokens, d]
    q_in, k_in = bf16_dev(wide)[..., :128], bf16_dev(kt).transpose(0, 1)
    p = to_dev(np.stack([pos[0], pos[0] + 1], 1).reshape(-1))[::2]
    w = to_dev(np.stack([qw, qw], 1).reshape(-1).view(np.int16)).view(torch.bfloat16)[::2]
    q, k = K.qk_norm_rope(q_in, k_in, w, None, to_dev(table), p)
    same_bits(host_u16(q), O.f32_to_bf16(KO.norm_rope(wide[..., :128], qw, table, pos)), "q")
    same_bits(host_u16(k), O.f32_to_bf16(KO.norm_rope(kt.transpose(1, 0, 2), None, table, pos)), "k")
    flat = bits(rng, 10 * 4 * 128 + 3)
    odd = bf16_dev(flat)[3:].view(10, 4, 128)           # 6 bytes off
    one = bits(rng, 1, 2, 128)
    q, k = K.qk_norm_rope(odd, bf16_dev(one).expand(10, 2, 128), bf16_dev(qw), bf16_dev(kw),
                          to_dev(table), to_dev(pos[0]))
    same_bits(host_u16(q), O.f32_to_bf16(KO.norm_rope(flat[3:].reshape(10, 4, 128), qw, table, pos)),
              "odd")
    same_bits(host_u16(k), O.f32_to_bf16(KO.norm_rope(np.repeat(one, 10, 0), kw, table, pos)),
              "broadcast")


def test_rope_special_values():
    """Zero, huge (the squares overflow), tiny, infinite and NaN heads stay in their own heads."""
    _, host, _, qw, kw, table, pos, _ = case(9, 6, 4, 1, 128, 64)
    q, k = host[0].copy(), host[1].copy()
    for t, v in enumerate((0.0, 1e30, 1e-30, np.inf, np.nan)):
        q[t, t % 4, 5] = O.f32_to_bf16(np.array([v], np.float32))[0]
        if t < 3:
            q[t, t % 4] = q[t, t % 4, 5]
    got, gk = K.qk_norm_rope(bf16_dev(q), bf16_dev(k), bf16_dev(qw), bf16_dev(kw), to_dev(table),
                             to_dev(pos[0]))
    same_bits(host_u16(got), O.f32_to_bf16(KO.norm_rope(q, qw, table, pos)), "q")
    same_bits(host_u16(gk), O.f32_to_bf16(KO.norm_rope(k, kw, table, pos)), "k")


def test_positions_outside_the_table_are_nan():
    _, host, dev, qw, kw, table, pos, axis = case(10, 12, 4, 2, 128, 64, 3)
    pos[0, 2], pos[1, 5], pos[2, 7] = -1, ROWS, 1 << 40
    axis[3] = 7
    q, _ = K.qk_norm_rope(dev[0], dev[1], bf16_dev(qw), bf16_dev(kw), to_dev(table), to_dev(pos),
                          axis=to_dev(axis))
    want = O.f32_to_bf16(KO.norm_rope(host[0], qw, table, pos, axis))
    same_bits(host_u16(q), want, "q")
    assert np.isnan(O.bf16_to_f32(want)).any() and not np.isnan(O.bf16_to_f32(want)).all()


def append_case(seed, T, Hq, Hkv, d, rot, page, pages, slots, axes=1, adjacent=False, edit=None):
    rng, host, dev, qw, kw, table, pos, axis = case(seed, T, Hq, Hkv, d, rot, axes)
    if edit:
        edit(host)
        dev = [bf16_dev(np.ascontiguousarray(h)) for h in host]
    before = rng.integers(0, 256, (pages, Hkv, page // 16, 17 * d), dtype=np.uint8)
    cache = to_dev(before)
    q = K.qk_norm_rope_append(*dev, bf16_dev(qw), bf16_dev(kw),
                              None if table is None else to_dev(table), dev_pos(pos), cache,
                              to_dev(np.asarray(slots, np.int64)),
                              axis=None if axis is None else to_dev(axis), adjacent=adjacent)
    want = before.copy()
    k = KO.norm_rope(host[1], kw, table, pos, axis, adjacent=adjacent)
    KO.write(want, slots, k, O.bf16_to_f32(host[2]))
    same_bits(host_u16(q), O.f32_to_bf16(KO.norm_rope(host[0], qw, table, pos, axis,
                                                      adjacent=adjacent)), "q")
    got = host_u8(cache)
    bad = np.argwhere(got != want)
    assert bad.size == 0, f"{len(bad)} cache bytes differ, first at {bad[:4].tolist()}"


@pytest.mark.parametrize("T,Hq,Hkv,d,rot,page,axes,adjacent", [
    (1, 32, 8, 128, 128, 16, 1, False), (5, 2, 2, 64, 64, 16, 1, False), (37, 8, 8, 64, 32, 32, 3, True),
    (19, 6, 2, 256, 64, 64, 3, False), (200, 12, 4, 128, 128, 128, 1, False),
    (41, 4, 1, 256, 256, 256, 1, True), (64, 3, 3, 128, 0, 16, 1, False)])
@pytest.mark.parametrize("chunk", [False, True])
def test_append_bytes(T, Hq, Hkv, d, rot, page, axes, adjacent, chunk):
    """Scattered slots, and a chunk through shuffled pages from the middle of one on; every other
    byte of the cache stays."""
    rng = np.random.default_rng(T)
    pages = -(-T // page) + 3
    if chunk:
        order = rng.permutation(pages)
        at = np.arange(T) + 5
        slots = order[at // page] * page + at % page
    else:
        slots = rng.permutation(pages * page)[:T]
    append_case(T + d, T, Hq, Hkv, d, rot, page, pages, slots, axes, adjacent)


def test_append_skips_slots_outside_the_cache():
    slots = np.array([-1, 3, 48, 47, -(1 << 40), 1 << 40, 0, 16 * (1 << 33), 31])
    append_case(3, 9, 4, 2, 128, 128, 16, 3, slots)


def test_append_special_values():
    """Blocks of zeros, of one tiny or huge value, at the scale's thresholds and rounding ties, NaN and
    infinity: the values' codes come straight from the inputs."""
    def edit(host):
        v = O.bf16_to_f32(host[2]).copy()
        v[0] = 0.0
        v[1, 0] = np.linspace(-7, 7, v.shape[2])
        v[2, 0, :32] = [7.0, 7.03125, -5, 5, 2.5, 3.5, 0.25, 0.75, 1.25, 1.75, -0.0] + [0.1] * 21
        v[2, 1, :32] = 7.03125
        v[3, 0, 40] = np.nan
        v[3, 1, 70] = np.inf
        v[4, 0] = 3e38
        v[4, 1] = 1e-38
        v[5, 0, 3], v[5, 1, 3] = 3.3e38, -1e-40
        host[2] = O.f32_to_bf16(v)
        k = host[1].copy()
        k[3, 0, 9] = 0x7FC0
        k[4, 1, 100] = 0x7F80
        k[5, 0] = 0
        host[1] = k
    append_case(4, 6, 4, 2, 128, 64, 16, 2, np.arange(6) * 3, edit=edit)


@pytest.mark.parametrize("T", [0, 1])
def test_zero_and_one_token(T):
    cache = K.new_cache(2, 2, 16, 128)
    z = lambda h: torch.zeros((T, h, 128), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = torch.zeros(T, dtype=torch.int64, device="cuda")
    q, k = K.qk_norm_rope(z(4), z(2), None, None, to_dev(angles(4, 64)), i)
    assert q.shape == (T, 4, 128) and k.shape == (T, 2, 128)
    q = K.qk_norm_rope_append(z(4), z(2), z(2), None, None, None, None, cache, i)
    assert q.shape == (T, 4, 128) and not q.any()
    k, v = K.gather(cache, i)
    assert k.shape == v.shape == (T, 2, 128) and not k.any() and not v.any()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (256, 128)])
def test_gather_reads_what_the_cache_holds(d, page):
    rng = np.random.default_rng(d)
    cache = rng.integers(0, 256, (5, 3, page // 16, 17 * d), dtype=np.uint8)
    s = cache[..., 16 * d:]
    s[:] = np.where(rng.random(s.shape) < 0.02, 255, s % 240 + 5)
    slots = np.concatenate([rng.permutation(5 * page)[:40], [-1, 5 * page, -(1 << 40), 1 << 40]])
    k, v = K.gather(to_dev(cache), to_dev(slots))
    wk, wv = KO.read(cache, slots)
    for got, want in ((k, wk), (v, wv)):
        g = O.bf16_to_f32(host_u16(got)).astype(np.float64)
        assert np.array_equal(g, want, equal_nan=True)


def test_append_into_a_layer_of_a_larger_cache():
    """The layers of a page side by side: a layer's pages are strided."""
    rng, host, dev, qw, kw, table, pos, _ = case(11, 20, 4, 2, 128, 128)
    whole = torch.zeros((6, 3, 2, 2, 17 * 128), dtype=torch.uint8, device="cuda")   # [pages, layers, ...]
    slots = rng.permutation(6 * 32)[:20]
    K.qk_norm_rope_append(*dev, bf16_dev(qw), bf16_dev(kw), to_dev(table), to_dev(pos[0]),
                          whole[:, 1], to_dev(slots))
    want = np.zeros((6, 2, 2, 17 * 128), np.uint8)
    KO.write(want, slots, KO.norm_rope(host[1], kw, table, pos), O.bf16_to_f32(host[2]))
    assert np.array_equal(host_u8(whole[:, 1]), want)
    assert not whole[:, 0].any() and not whole[:, 2].any()
    k, _ = K.gather(whole[:, 1], to_dev(slots))
    assert np.array_equal(O.bf16_to_f32(host_u16(k)), KO.read(want, slots)[0].astype(np.float32))
