"""K.sample_tokens against the definition in 64 bits: the same ids.

A draw whose border lies within 1e-9 of the row's weight could go either way
(weights are held to 3e-13 of the best, sums of 2^18 of them to 2^-27 at worst);
the tests' draws do not come that near."""
import math

import numpy as np
import pytest
import torch

from moc_amd import _native as N
from moc_amd import kernels as K

import paged_reference as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = x.shape[0]
    dev = lambda t, dt: t if not isinstance(t, list) else torch.tensor(t, dtype=dt, device="cuda")  # noqa: E731
    got = K.sample_tokens(x, torch.tensor(u, dtype=F32, device="cuda"), dev(temperature, F32), dev(top_k, torch.int32),
                          dev(top_p, F32), dev(min_p, F32)).tolist()
    xs = x.float().cpu().numpy()
    f32 = lambda t, r: float(np.float32(t[r] if isinstance(t, list) else t))  # noqa: E731
    for r in range(rows):
        k = top_k[r] if isinstance(top_k, list) else top_k
        want, near = R.sample(xs[r], f32(u, r), f32(temperature, r), k, f32(top_p, r), f32(min_p, r))
        assert got[r] == want or near < 1e-9, (r, got[r], want, near)
    return got


def _logits(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype).cuda()


def _u(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=500, top_p=0.9), dict(top_p=0.1),
            dict(top_p=0.95, temperature=1.3), dict(min_p=0.05), dict(top_k=40, top_p=0.8, min_p=0.1, temperature=0.9),
            dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0), dict(min_p=2.0), dict(temperature=50.0, top_p=0.999),
            dict(temperature=1e-3), dict(temperature=-1.0, top_k=3)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda d: "-".join("%s%g" % i for i in d.items()) or "plain")
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [1000, 32000])
def test_against_the_definition(settings, dtype, vocab):
    _check(_logits(8, vocab, dtype, vocab), _u(8, 3), **settings)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1023, 1024, 1025, 5461, 50257, 128256, 262144])
def test_vocabularies(dtype, vocab):
    x = _logits(3, vocab, dtype, vocab)
    _check(x, _u(3, vocab), top_k=[0, 5, 2000], top_p=[0.9, 1.0, 0.97], temperature=[1.0, 0.8, 1.5])
    _check(x, _u(3, vocab + 1))


def test_every_word_can_be_drawn():
    """u across [0, 1): each word for the share of u that is its weight."""
    x = _logits(1, 40, F32, 5, 1.0).expand(2000, 40)
    u = [(i + 0.5) / 2000 for i in range(2000)]
    got = np.array(_check(x, u))
    w = torch.softmax(x[0].double(), 0).cpu().numpy()
    assert (np.abs(np.bincount(got, minlength=40) / 2000 - w) <= 1.0 / 2000 + 1e-12).all()
    assert (np.diff(got) >= 0).all()


def test_rows_have_their_own_settings():
    rows = 64
    g = torch.Generator().manual_seed(8)
    r = torch.rand(4, rows, generator=g)
    _check(_logits(rows, 9001, F32, 8), _u(rows, 9), temperature=(r[0] * 1.5 - 0.1).tolist(),
           top_k=(r[1] * 200 - 50).int().tolist(), top_p=(r[2] * 1.1).tolist(), min_p=(r[3] * 0.2 - 0.05).tolist())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_equal_logits(dtype):
    """Ties go to the lower id, across the whole row and at each rule's border."""
    x = torch.zeros(6, 3001, dtype=dtype, device="cuda")
    got = _check(x, [0.0, 0.5, 0.999, 0.3, 0.3, 0.9], top_k=[0, 0, 0, 10, 0, 0], top_p=[1.0, 1.0, 1.0, 1.0, 0.01, 0.5])
    assert got[3] == 3 and got[4] < 31 and got[5] < 1501
    x[:, ::3] = -0.0
    assert _check(x, [0.0, 0.5, 0.999, 0.3, 0.3, 0.9], top_k=[0, 0, 0, 10, 0, 0],
                  top_p=[1.0, 1.0, 1.0, 1.0, 0.01, 0.5]) == got
    y = _logits(6, 3001, dtype, 4).mul_(2).round_().div_(2)  # few distinct values
    for top_k in (1, 7, 100, 2999, 3001, 5000):
        _check(y, _u(6, top_k), top_k=top_k)
        _check(y, _u(6, top_k), top_k=top_k, top_p=0.6)
    assert K.sample_tokens(y, torch.zeros(6, device="cuda"), 0.0).tolist() == [
        int(np.argmax(r)) for r in y.float().cpu().numpy()]


def test_masked_words():
    """-infinity, the type's lowest value, NaN, +infinity."""
    x = _logits(8, 5000, F32, 6)
    x[0, 100:] = -math.inf
    x[1, :] = -math.inf
    x[1, 4321] = -7.0
    x[2, :4999] = torch.finfo(F32).min
    x[3, 17], x[3, 4000] = math.inf, math.inf
    x[4, ::2] = math.nan
    x[5, :] = torch.finfo(F32).min
    x[6, :], x[7, :] = -math.inf, math.nan
    for more in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                 dict(top_k=200, top_p=0.5, min_p=0.01)):
        got = _check(x, _u(8, 7), **more)
        assert got[1] == 4321 and got[2] == 4999 and got[3] in (17, 4000) and got[4] % 2 and got[6] == got[7] == -1


def test_ends_of_u():
    """0: the first word with weight; 1 and more, and NaN (as 0): still a word with weight."""
    x = _logits(1, 300, F32, 2).repeat(5, 1)
    x[:, :10] = -math.inf
    x[:, 290:] = -math.inf
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, math.nan], device="cuda")
    assert K.sample_tokens(x, u).tolist() == [10, 289, 289, 10, 10]


def test_strides_and_streams():
    wide = _logits(6, 4000, F32, 3)
    u = torch.tensor(_u(6, 1), device="cuda")
    want = K.sample_tokens(wide[:, 8:3009].contiguous(), u, top_p=0.9)
    assert torch.equal(K.sample_tokens(wide[:, 8:3009], u, top_p=0.9), want)
    assert torch.equal(K.sample_tokens(wide[:, 8:3009].t().contiguous().t(), u, top_p=0.9), want)
    assert torch.equal(K.sample_tokens(wide[:, 7:3008], u, top_p=0.9), K.sample_tokens(wide[:, 7:3008].clone(), u, top_p=0.9))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(K.sample_tokens(wide[:, 8:3009], u, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)


def test_no_rows():
    assert K.sample_tokens(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


@pytest.mark.parametrize("rows", [1, 40])
def test_graph_replays(rows):
    """New logits, numbers and settings in the captured buffers."""
    x, u = _logits(rows, 32000, F32, 1), torch.zeros(rows, device="cuda")
    t, k = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    p, m = torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda")
    K.sample_tokens(x, u, t, k, p, m)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.sample_tokens(x, u, t, k, p, m)
    for i in range(6):
        x.copy_(_logits(rows, 32000, F32, 50 + i))
        u.copy_(torch.tensor(_u(rows, i)))
        k.fill_((0, 50, 3)[i % 3])
        p.fill_((0.9, 1.0, 0.5)[i // 2])
        t.fill_((1.0, 0.0, 0.7)[i % 3])
        want = K.sample_tokens(x, u, t, k, p, m)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want)
        for r in range(0, rows, 13):
            id_, near = R.sample(x[r].cpu().numpy(), float(u[r]), float(t[r]), int(k[r]), float(p[r]), 0.0)
            assert int(out[r]) == id_ or near < 1e-9


# ---------------------------------------- rows spread over several workgroups
def _alone(x, u, temperature, top_k, top_p, min_p):
    """The form of one workgroup a row, which takes no workspace."""
    out = torch.empty(x.shape[0], dtype=torch.int64, device="cuda")
    N.call("moc_sample_tokens", N.dtype_code(x.dtype), x.data_ptr(), *x.shape, x.stride(0), u.data_ptr(),
           temperature.data_ptr(), 0.0, top_k.data_ptr(), 0, top_p.data_ptr(), 0.0, min_p.data_ptr(), 0.0, out.data_ptr(),
           torch.cuda.current_stream().cuda_stream)
    return out


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda d: "-".join("%s%g" % i for i in d.items()) or "plain")
@pytest.mark.parametrize("dtype,vocab", [(F32, 65536), (BF, 128256), (F32, 70001), (BF, 100001)])
def test_long_rows_against_the_definition(settings, dtype, vocab):
    _check(_logits(4, vocab, dtype, vocab + 1), _u(4, 5), **settings)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,vocab", [(1, 262144), (7, 49152), (33, 65537), (64, 50257), (300, 66000)])
def test_long_rows_equal_one_workgroup(dtype, rows, vocab):
    """Bit for bit, over mixed settings and rows of every kind: equal words, NaN and
    infinities, all masked, one word alone, a few words over a masked row."""
    x = _logits(rows, vocab, dtype, rows)
    kinds = torch.arange(rows) % 8
    for r in range(rows):
        kind = int(kinds[r]) if rows > 1 else 0
        if kind == 1:
            x[r] = 1.5
        elif kind == 2:
            x[r, ::97] = math.nan
            x[r, 5::1009] = math.inf
        elif kind == 3:
            x[r] = -math.inf
        elif kind == 4:
            x[r] = torch.finfo(dtype).min
            x[r, [3, vocab // 2, vocab - 1]] = 2.0
        elif kind == 5:
            x[r] = (x[r] * 2).round() / 2
        elif kind == 6:
            x[r, 1:] = -math.inf
    g = torch.Generator().manual_seed(rows)
    u = torch.rand(rows, generator=g).cuda()
    pick = lambda values, dt: torch.tensor(values, dtype=dt)[torch.randint(len(values), (rows,), generator=g)].cuda()  # noqa: E731
    for _ in range(6):
        s = (pick([1.0, 0.6, 1.7, 0.0, 30.0], F32), pick([0, 0, 0, 3, 700], torch.int32), pick([1.0, 0.95, 0.5, 1e-6, 0.9999], F32),
             pick([0.0, 0.0, 0.02, 1.0], F32))
        assert torch.equal(K.sample_tokens(x, u, *s), _alone(x, u, *s))


def test_long_rows_strided_and_replayed():
    """Rows off the 16-byte grid; a captured call follows its inputs, with its own
    workspace, beside an eager one."""
    wide = _logits(3, 70003, F32, 9)
    x = wide[:, 1:70000]
    u = torch.tensor([0.1, 0.5, 0.9], device="cuda")
    full = lambda v, dt=F32: torch.full((3,), v, dtype=dt, device="cuda")  # noqa: E731
    s = (full(1.0), full(0, torch.int32), full(0.9), full(0.0))
    K.sample_tokens(x, u, *s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.sample_tokens(x, u, *s)
    for i in range(4):
        wide.copy_(_logits(3, 70003, F32, 20 + i))
        u.copy_(torch.tensor(_u(3, i), device="cuda"))
        graph.replay()
        eager = K.sample_tokens(x, u, *s)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(eager, _alone(x, u, *s)), i
