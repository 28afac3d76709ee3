"""The gated delta rule on the GPU against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from tests._check import bf16_dev, to_dev
from tests._decode import Delta, host, i32, same, starts_of
from vllm_sly_radiance_amd import _native_decode
from vllm_sly_radiance_amd import radiance_gdn as G

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_decode.lib()


HEADS = [(2, 6, 128, 128), (2, 2, 64, 64), (1, 4, 64, 128), (3, 3, 128, 64)]
LENS = [[1], [1] * 9, [5, 8, 1, 3], [16, 17], [31, 0, 33], [63, 64, 65], [1, 300, 2, 128, 129, 0]]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_against_the_definition(heads, lens):
    d = Delta(np.random.default_rng(len(lens) + sum(lens) + heads[1]), lens, heads)
    args = d.device()
    d.check(G.gated_delta_rule(*args), args[7])


@pytest.mark.parametrize("lens", [[4], [1, 37, 20], [100, 2]], ids=str)
@pytest.mark.parametrize("max_q", [1, 16, 17, 4096])
def test_max_q_is_only_a_hint(lens, max_q):
    d = Delta(np.random.default_rng(3), lens, (1, 2, 128, 128))
    args = d.device(max_q=max_q)
    d.check(G.gated_delta_rule(*args), args[7])


@pytest.mark.parametrize("lens,cols", [([8, 8], 8), ([5, 1, 0, 3], 5), ([3, 40], 4), ([70, 1], 2)])
def test_the_state_after_each_token(lens, cols):
    d = Delta(np.random.default_rng(8), lens, (2, 4, 128, 128), slots=len(lens) * cols + 3)
    write = np.random.default_rng(9).permutation(d.slots)[:len(lens) * cols].reshape(len(lens), cols)
    d.read = write[:, -1].astype(np.int32)          # as after a step whose last token was accepted
    args = d.device(write)
    d.check(G.gated_delta_rule(*args), args[7], write)


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [30, 70, 9, 64]], ids=str)
def test_slots(lens):
    """New sequences, forks (read here, written there), sequences whose state nobody wants, slots past the
    pool."""
    d = Delta(np.random.default_rng(4), lens, (1, 3, 128, 128), slots=7, read=[-1, 5, 2, 9])
    write = np.array([3, 6, -1, 7], np.int32)
    args = d.device(write)
    out = host(G.gated_delta_rule(*args))
    ref, tol, states, bounds = d.expect()
    n = sum(lens[:3])
    assert (np.abs(out[:n] - ref[:n]) <= tol[:n]).all() and np.isnan(out[n:]).all()
    got = host(args[7])
    for b, s in ((0, 3), (1, 6)):
        assert (np.sqrt(((got[s] - states[b][-1]) ** 2).sum(1)) <= bounds[b][-1]).all()
    for s in (0, 1, 2, 4, 5):
        assert np.array_equal(got[s], d.state[s])


def test_a_sequence_without_tokens_hands_its_state_on():
    d = Delta(np.random.default_rng(5), [0, 2, 0, 0], (1, 2, 64, 64), slots=6, read=[1, 1, -1, 8])
    write = np.array([0, 2, 3, 4], np.int32)
    for max_q in (2, 100):
        args = d.device(write, max_q)
        G.gated_delta_rule(*args)
        got = args[7].cpu().numpy()
        assert np.array_equal(got[0], d.state[1]) and not got[3].any() and np.isnan(got[4]).all()
        assert np.array_equal(got[1], d.state[1]) and np.array_equal(got[5], d.state[5])


@pytest.mark.parametrize("lens", [[1, 2], [65, 3]], ids=str)
def test_rows_of_no_sequence_stay(lens):
    d = Delta(np.random.default_rng(6), lens, (1, 2, 128, 128), extra_rows=5)
    args = d.device()
    want = G.gated_delta_rule(*args)
    shift = d.device()
    for i in range(5):                  # rows before the first sequence as well
        shift[i] = torch.cat([shift[i][-2:], shift[i][:-2]])
    shift[8] = shift[8] + 2
    out = G.gated_delta_rule(*shift)
    n = sum(lens)
    assert torch.equal(out[2:2 + n], want[:n]) and same(shift[7], args[7])


@pytest.mark.parametrize("lens", [[3, 2], [40, 90]], ids=str)
def test_views_and_strides(lens):
    """Heads inside a wider projection, gates side by side, states of one layer of several, and layouts that
    are copied first."""
    Hk, Hv, dk, dv = heads = (2, 4, 128, 64)
    d = Delta(np.random.default_rng(7), lens, heads)
    args = d.device()
    want = G.gated_delta_rule(*args)
    T = sum(lens)
    wide = torch.full((T, 2 * Hk * dk + Hv * dv + 24), 9.0, dtype=torch.bfloat16, device="cuda")
    q, k, v = (wide[:, 8:8 + Hk * dk].unflatten(1, (Hk, dk)),
               wide[:, 8 + Hk * dk:8 + 2 * Hk * dk].unflatten(1, (Hk, dk)),
               wide[:, 8 + 2 * Hk * dk:8 + 2 * Hk * dk + Hv * dv].unflatten(1, (Hv, dv)))
    gates = torch.zeros((T, 2 * Hv + 1), dtype=torch.bfloat16, device="cuda")
    state = torch.zeros((d.slots, 3, Hv, dk, dv), device="cuda")
    for x, y in ((q, 0), (k, 1), (v, 2), (gates[:, :Hv], 3), (gates[:, Hv + 1:], 4)):
        x.copy_(d.device()[y])
    state[:, 1] = d.device()[7]
    new = d.device()
    new[:5] = [q, k, v, gates[:, :Hv], gates[:, Hv + 1:]]
    new[7] = state[:, 1]
    assert torch.equal(G.gated_delta_rule(*new), want) and torch.equal(state[:, 1], args[7])
    assert not state[:, 0].any() and not state[:, 2].any()
    odd = d.device()
    odd[0] = odd[0].transpose(0, 1).contiguous().transpose(0, 1)
    odd[1] = torch.cat([odd[1], odd[1]], 2)[..., 4:4 + dk].copy_(odd[1])
    odd[2] = odd[2].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    odd[3] = odd[3].T.contiguous().T
    assert torch.equal(G.gated_delta_rule(*odd), want)


@pytest.mark.parametrize("lens", [[1], [6], [70, 130]], ids=str)
def test_decay_of_everything_and_of_nothing(lens):
    """Gates at infinity: a forgets the state (or nothing of it), b ignores the token (or takes it whole)."""
    from oracle import mxfp4_oracle as O
    d = Delta(np.random.default_rng(10), lens, (1, 2, 128, 128))
    rng = np.random.default_rng(11)
    for g in (d.a, d.b):
        x = O.bf16_to_f32(g).copy()
        for value in (np.inf, -np.inf, 300.0, -300.0):
            x[rng.random(x.shape) < 0.15] = value
        g[:] = O.f32_to_bf16(x)
    args = d.device()
    d.check(G.gated_delta_rule(*args), args[7])


@pytest.mark.parametrize("what", ["q", "k", "v", "a", "b"])
@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=str)
@pytest.mark.parametrize("lens,at", [([6, 3], 2), ([150, 20], 70)], ids=str)
def test_what_is_not_finite_reaches_no_one_earlier(what, bad, lens, at):
    """NaN in a query is its own token's; in a key, a value or a gate it is there from that token on, in the
    heads (for values: the channels) that have it, and in no other sequence."""
    heads = (2, 4, 128, 128)
    d = Delta(np.random.default_rng(12), lens, heads)
    want = d.expect()
    x = getattr(d, what)
    one = np.uint16(0x7FC0 if np.isnan(bad) else 0x7F80)
    if what in "qk":
        x[at, 1, 5] = one
        heads_hit, cols = [2, 3], slice(None)
    elif what == "v":
        x[at, 1, 7] = one
        heads_hit, cols = [1], slice(7, 8)
    else:
        if what == "b" or not np.isnan(bad):
            one = np.uint16(0x7FC0)             # (gates at infinity are meant)
        x[at, 3] = one
        heads_hit, cols = [3], slice(None)
    args = d.device()
    out, state = host(G.gated_delta_rule(*args)), host(args[7])
    hit = np.zeros(out.shape, bool)
    for h in heads_hit:
        hit[at:at + 1 if what == "q" else lens[0], h, cols] = True
    assert not np.isfinite(out[hit]).any()
    ref, tol, states, bounds = want
    assert (np.abs(out - ref)[~hit] <= tol[~hit]).all()
    for b in range(2):
        s = state[d.write[b]]
        off = np.sqrt(((s - states[b][-1]) ** 2).sum(1))
        fine = off <= bounds[b][-1]
        bad_state = np.zeros(fine.shape, bool)
        if b == 0 and what != "q":
            for h in heads_hit:
                bad_state[h, cols] = True
        assert (fine == ~bad_state).all()


@pytest.mark.parametrize("v_scale", [1e-30, 1e30])
def test_values_of_any_size(v_scale):
    d = Delta(np.random.default_rng(13), [90, 3], (1, 2, 128, 128), read=[-1, -1], v_scale=v_scale)
    args = d.device()
    ref, tol, states, bounds = d.expect()
    out = host(G.gated_delta_rule(*args))
    assert (np.abs(out - ref) <= tol).all()
    for b in range(2):
        off = np.sqrt(((host(args[7])[d.write[b]] - states[b][-1]) ** 2).sum(1))
        assert (off <= bounds[b][-1]).all()


@pytest.mark.parametrize("lens", [[40], [200]], ids=str)
def test_the_same_key_again_and_again(lens):
    """Every token with one key, beta near 1 and hardly any decay: the chunks' triangular systems at their worst
    conditioned."""
    from oracle import mxfp4_oracle as O
    d = Delta(np.random.default_rng(14), lens, (1, 2, 128, 128))
    d.k[:] = d.k[0]
    d.k[1::3] ^= 0x8000                 # and its negative
    d.b[:] = O.f32_to_bf16(np.full(d.b.shape, 6.0, np.float32))
    d.a[:] = O.f32_to_bf16(np.full(d.a.shape, -8.0, np.float32))
    args = d.device()
    d.check(G.gated_delta_rule(*args), args[7])


def test_scale_and_eps():
    d = Delta(np.random.default_rng(15), [70, 2], (1, 2, 64, 64))
    for kw in (dict(scale=0.5, eps=1e-2), dict(scale=-3.0, eps=0.0), dict(scale=0.0)):
        args = d.device()
        d.check(G.gated_delta_rule(*args, **kw), args[7], **kw)


def test_zero_keys_and_queries():
    """eps keeps what has no length from dividing by zero."""
    d = Delta(np.random.default_rng(16), [66, 2], (1, 2, 128, 128))
    d.k[3:50:7], d.q[5:60:6] = 0, 0
    args = d.device()
    d.check(G.gated_delta_rule(*args), args[7])


@pytest.mark.parametrize("lens", [[1] * 5, [70, 1, 200]], ids=str)
def test_captured(lens):
    """A graph replayed with other inputs, starts and slots in its buffers, eager work between, gives what
    eager calls give; twice at once with workspaces of their own."""
    d = Delta(np.random.default_rng(17), lens, (2, 4, 128, 128))
    eager, held = d.device(), d.device()
    twin = d.device()
    G.gated_delta_rule(*d.device())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.gated_delta_rule(*held)
        out2 = G.gated_delta_rule(*twin)
    held[7].copy_(eager[7]), twin[7].copy_(eager[7])
    for i in range(4):
        other = Delta(np.random.default_rng(30 + i), lens[::-1] if i % 2 else lens, (2, 4, 128, 128))
        src = other.device()
        for j in (0, 1, 2, 3, 4, 8, 9, 10):
            for x in (eager, held, twin):
                x[j].copy_(src[j])
        want = G.gated_delta_rule(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)
        assert torch.equal(held[7], eager[7]) and torch.equal(twin[7], eager[7])


def test_streams():
    """Calls on two streams at once, each on tensors of its own."""
    ds = [Delta(np.random.default_rng(20 + i), [100 + 50 * i, 3], (2, 4, 128, 128)) for i in range(2)]
    args = [d.device() for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    outs = []
    for a, s in zip(args, streams):
        with torch.cuda.stream(s):
            outs.append(G.gated_delta_rule(*a))
    torch.cuda.synchronize()
    for d, o, a in zip(ds, outs, args):
        d.check(o, a[7])


def test_a_step_is_a_prompt_cut_in_pieces():
    """A prompt in one call, and in calls of 1, 7, 64, 100 tokens that go on from each other."""
    d = Delta(np.random.default_rng(21), [172], (1, 2, 128, 128), read=[-1])
    args = d.device()
    whole = G.gated_delta_rule(*args)
    again = d.device()
    at = 0
    for n in (1, 7, 64, 100):
        part = [x[at:at + n] for x in again[:5]]
        read = i32([-1]) if at == 0 else again[10]
        out = G.gated_delta_rule(*part, *again[5:8], i32(starts_of([n])), read, again[10], n)
        ref, tol, *_ = d.expect()
        assert (np.abs(host(out) - ref[at:at + n]) <= tol[at:at + n]).all()
        at += n
    d.check(whole, args[7])
    d.check(whole, again[7])


def test_nothing_to_do():
    d = Delta(np.random.default_rng(22), [], (1, 2, 64, 64))
    args = d.device()
    assert G.gated_delta_rule(*args).shape == (0, 2, 64)
    d = Delta(np.random.default_rng(23), [0, 0], (1, 2, 64, 64))
    args = d.device()
    assert G.gated_delta_rule(*args).shape == (0, 2, 64)
    assert np.array_equal(args[7].cpu().numpy(), d.state)


def test_starts_out_of_range_stay_inside():
    """Starts past the rows, or negative, are held to them."""
    d = Delta(np.random.default_rng(24), [3, 70], (1, 2, 128, 128))
    args = d.device()
    args[8] = i32([-4, 3, 90])
    want = d.device()
    assert torch.equal(G.gated_delta_rule(*args), G.gated_delta_rule(*want))
    assert same(args[7], want[7])


def test_many_sequences():
    """More sequences than a wave has lanes, of uneven lengths."""
    rng = np.random.default_rng(25)
    lens = rng.integers(0, 40, 150).tolist()
    lens[77] = 333
    d = Delta(rng, lens, (1, 1, 64, 64))
    args = d.device()
    d.check(G.gated_delta_rule(*args), args[7])


REFUSED = [
    (dict(q=lambda a: a[0].float()), "q must be bf16"),
    (dict(k=lambda a: a[1][:, :1]), "k must be bf16 .3, 2, 128."),
    (dict(v=lambda a: a[2][:2]), "v must be bf16 .3, 4, 128."),
    (dict(q=lambda a: a[0][..., :96], k=lambda a: a[1][..., :96]), "state must be fp32|none of 64, 128"),
    (dict(a=lambda a: a[3].float()), "a must be bf16"),
    (dict(b=lambda a: a[4][:, :3]), "b must be bf16"),
    (dict(a_log=lambda a: a[5].double()), "a_log must be fp32"),
    (dict(dt_bias=lambda a: a[6][:3]), "dt_bias must be fp32"),
    (dict(state=lambda a: a[7].bfloat16()), "state must be fp32"),
    (dict(state=lambda a: a[7].transpose(2, 3)), "contiguous"),
    (dict(state=lambda a: a[7][:, :2]), "state must be fp32"),
    (dict(q_starts=lambda a: a[8][:2]), "q_starts must be int32 .3."),
    (dict(q_starts=lambda a: a[8].long()), "q_starts must be int32"),
    (dict(read_slots=lambda a: a[9].long()), "read_slots must be int32"),
    (dict(write_slots=lambda a: a[10][:1]), "write_slots must be int32"),
    (dict(write_slots=lambda a: a[10].view(2, 1)[:, :0]), "no columns"),
    (dict(max_q=lambda a: -1), "max_q=-1"),
    (dict(scale=lambda a: float("nan")), "scale is NaN"),
    (dict(eps=lambda a: -1.0), "eps"),
    (dict(b=lambda a: a[4].cpu()), "cuda:0 and cpu"),
    (dict(max_q=lambda a: 1 << 40), "out of range"),
]


@pytest.mark.parametrize("change,words", REFUSED, ids=lambda x: "-".join(x) if isinstance(x, dict) else "")
def test_refused(change, words):
    names = ["q", "k", "v", "a", "b", "a_log", "dt_bias", "state", "q_starts", "read_slots", "write_slots", "max_q"]
    d = Delta(np.random.default_rng(26), [1, 2], (2, 4, 128, 128))
    args = d.device()
    kw = dict(zip(names, args))
    kw.update({n: f(args) for n, f in change.items()})
    with pytest.raises(RuntimeError, match=words):
        G.gated_delta_rule(**kw)
    d.check(G.gated_delta_rule(*args), args[7])         # and the next call is served


def test_gradients_are_refused_and_writes_count():
    d = Delta(np.random.default_rng(27), [2], (1, 2, 64, 64))
    args = d.device()
    before = args[7]._version
    G.gated_delta_rule(*args)
    assert args[7]._version > before
    args[2].requires_grad_()
    with pytest.raises(RuntimeError):
        G.gated_delta_rule(*args).sum().backward()


def test_new_state():
    s = G.new_state(3, 4, 128, 64, layers=2)
    assert s.shape == (2, 3, 4, 128, 64) and s.dtype == torch.float32 and not s.any()
    with pytest.raises(RuntimeError, match="none of"):
        G.new_state(3, 4, 96, 64)
    with pytest.raises(RuntimeError, match="width"):
        G.new_conv_state(3, 64, 5)
    assert bf16_dev(np.zeros(2, np.uint16)).dtype == torch.bfloat16 and to_dev(np.zeros(1)).is_cuda
