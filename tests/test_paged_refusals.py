"""What K.paged_kv, K.paged_append, K.paged_attention and K.sample_tokens refuse,
and the C entries behind them, without a device: nothing is launched."""
import ctypes

import pytest
import torch

from moc_amd import _native as N
from moc_amd import kernels as K

BF, E4, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


@pytest.fixture
def calls(monkeypatch):
    """CPU tensors taken for device tensors; the calls that reach the library."""
    seen = []
    monkeypatch.setattr(N, "require_device", lambda *t: None)
    monkeypatch.setattr(N, "stream_on", lambda d: 0)
    monkeypatch.setattr(N, "is_current", lambda d: True)
    monkeypatch.setattr(N, "call", lambda name, *a: seen.append((name, a)))
    return seen


def _kv(**change):
    t = dict(k=torch.zeros(6, 2, 16, 64, dtype=torch.uint8).view(E4), v=torch.zeros(6, 2, 16, 64, dtype=torch.uint8).view(E4),
             k_scale=torch.zeros(6, 2), v_scale=torch.zeros(6, 2))
    return K.PagedKV(**{**t, **change})


def _args(**change):
    t = dict(q=torch.zeros(3, 4, 64, dtype=BF), k=torch.zeros(3, 2, 64, dtype=BF), v=torch.zeros(3, 2, 64, dtype=BF),
             cos=torch.zeros(40, 32), sin=torch.zeros(40, 32), kv=_kv(), table=torch.zeros(3, 2, dtype=I32),
             lens=torch.zeros(3, dtype=I32))
    return {**t, **change}


def _attention(a):
    return {n: a[n] for n in a if n not in ("k", "v", "cos", "sin")}


BOTH = [
    ("q of f32", dict(q=torch.zeros(3, 4, 64))),
    ("q of two dimensions", dict(q=torch.zeros(3, 256, dtype=BF))),
    ("q of another head size", dict(q=torch.zeros(3, 4, 128, dtype=BF))),
    ("codes of another type", dict(kv=_kv(k=torch.zeros(6, 2, 16, 64, dtype=torch.uint8)))),
    ("codes of two types", dict(kv=_kv(v=torch.zeros(6, 2, 16, 64, dtype=torch.int8)))),
    ("scales of bf16", dict(kv=_kv(k_scale=torch.zeros(6, 2, dtype=BF)))),
    ("scales of another shape", dict(kv=_kv(v_scale=torch.zeros(6, 1)))),
    ("caches of two shapes", dict(kv=_kv(v=torch.zeros(5, 2, 16, 64, dtype=torch.uint8).view(E4)))),
    ("a cache that is a view", dict(kv=_kv(k=torch.zeros(6, 2, 16, 128, dtype=torch.uint8).view(E4)[..., :64]))),
    ("int64 lengths", dict(lens=torch.zeros(3, dtype=torch.int64))),
    ("an int64 table", dict(table=torch.zeros(3, 2, dtype=torch.int64))),
    ("a table of too few rows", dict(table=torch.zeros(2, 2, dtype=I32))),
    ("a table of columns", dict(table=torch.zeros(2, 3, dtype=I32).t())),
    ("lengths of too many sequences", dict(lens=torch.zeros(4, dtype=I32), table=torch.zeros(4, 2, dtype=I32))),
    ("lengths with a stride", dict(lens=torch.zeros(6, dtype=I32)[::2])),
    ("int64 cu", dict(cu=torch.zeros(4, dtype=torch.int64))),
    ("cu of another length", dict(cu=torch.zeros(3, dtype=I32))),
    ("out of another shape", dict(out=torch.zeros(3, 2, 64, dtype=BF))),
    ("out of f32", dict(out=torch.zeros(3, 4, 64))),
    ("out whose rows overlap", dict(out=torch.zeros(1, 4, 64, dtype=BF).expand(3, 4, 64))),
    ("out off the 16-byte grid", dict(out=torch.zeros(3 * 4 * 64 + 1, dtype=BF)[1:].view(3, 4, 64))),
]


@pytest.mark.parametrize("what,change", BOTH, ids=[w for w, _ in BOTH])
def test_both_refuse(calls, what, change):
    a = _args(**change)
    with pytest.raises(ValueError):
        K.paged_append(**a)
    with pytest.raises(ValueError):
        K.paged_attention(**_attention(a))
    assert not calls


def test_both_take(calls):
    a = _args()
    assert K.paged_append(**a).shape == (3, 4, 64) and K.paged_attention(**_attention(a)).shape == (3, 4, 64)
    cu = torch.tensor([0, 1, 1], dtype=I32)
    a = _args(cu=cu, lens=torch.zeros(2, dtype=I32), table=torch.zeros(2, 2, dtype=I32))
    K.paged_append(**a)
    K.paged_attention(**_attention(a))
    assert [n for n, _ in calls] == ["moc_paged_append_bf16", "moc_paged_attention_bf16"] * 2


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(3, 4, 64, dtype=BF)), dict(v=torch.zeros(2, 2, 64, dtype=BF)), dict(k=torch.zeros(3, 2, 64)),
    dict(v=torch.zeros(3, 2, 64)), dict(cos=torch.zeros(40, 64)), dict(sin=torch.zeros(39, 32)),
    dict(sin=torch.zeros(40, 32, dtype=BF)), dict(cos=torch.zeros(40, 32).half(), sin=torch.zeros(40, 32).half()),
    dict(cos=torch.zeros(32, 40).t(), sin=torch.zeros(32, 40).t())])
def test_append_refuses(calls, change):
    with pytest.raises(ValueError):
        K.paged_append(**_args(**change))
    assert not calls


def test_attention_refuses_heads_that_do_not_divide(calls):
    for heads in (0, 3, 5):
        with pytest.raises(ValueError):
            K.paged_attention(**_attention(_args(q=torch.zeros(3, heads, 64, dtype=BF))))


@pytest.mark.parametrize("bad", [dict(page=24), dict(page=8), dict(page=512), dict(head_dim=96), dict(kv_heads=0),
                                 dict(pages=-1), dict(dtype=BF)])
def test_cache_refuses(bad):
    with pytest.raises(ValueError):
        K.paged_kv(**{**dict(pages=2, kv_heads=1, page=16, head_dim=64, device="cpu"), **bad})
    kv = K.paged_kv(2, 1, 16, 64, device="cpu")
    assert kv.k.dtype == E4 and kv.k.shape == (2, 1, 16, 64) and kv.v_scale.shape == (2, 1)


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(3, 50).half()), dict(logits=torch.zeros(150)), dict(u=torch.zeros(2)),
    dict(u=torch.zeros(3, dtype=torch.float64)), dict(temperature=torch.ones(2)), dict(top_k=torch.ones(3)),
    dict(top_k=torch.ones(3, dtype=torch.int64)), dict(top_p=torch.ones(3, dtype=BF)), dict(min_p=torch.ones(3, 1)),
    dict(u=torch.zeros(6)[::2]), dict(min_p=torch.zeros(6)[::2])])
def test_sample_refuses(calls, change):
    with pytest.raises(ValueError):
        K.sample_tokens(**{**dict(logits=torch.zeros(3, 50), u=torch.zeros(3)), **change})
    assert not calls


def test_host_tensors_are_refused():
    a = _args()
    for call in (lambda: K.paged_append(**a), lambda: K.paged_attention(**_attention(a)),
                 lambda: K.sample_tokens(torch.zeros(3, 50), torch.zeros(3))):
        with pytest.raises(ValueError, match="device tensors"):
            call()


# -------------------------------------------------------------- the C entries
P = ctypes.c_void_p(1 << 20)


def _c_append(**c):
    d = dict(q=P, q_ld=256, q_lh=64, k=P, k_ld=128, k_lh=64, v=P, v_ld=128, v_lh=64, tokens=3, heads=4, kv_heads=2, dim=64,
             cos=P, sin=P, table_dtype=N.MOC_F32, angles=40, code=N.MOC_E4M3, kc=P, vc=P, ks=P, vs=P, pages=6, page=16,
             table=P, ld_table=2, width=2, lens=P, cu=None, seqs=3, out=P, o_ld=256, o_lh=64, stream=None)
    return N.load().moc_paged_append_bf16(*{**d, **c}.values())


def _c_attention(**c):
    d = dict(q=P, q_ld=256, q_lh=64, tokens=3, heads=4, kv_heads=2, dim=64, code=N.MOC_E4M3, kc=P, vc=P, ks=P, vs=P, pages=6,
             page=16, table=P, ld_table=2, width=2, lens=P, cu=None, seqs=3, scale=0.125, out=P, o_ld=256, o_lh=64, ws=None,
             bytes=0, stream=None)
    return N.load().moc_paged_attention_bf16(*{**d, **c}.values())


def _c_sample(**c):
    d = dict(dtype=N.MOC_F32, x=P, rows=2, vocab=50, ld=50, u=P, t=None, t1=1.0, k=None, k1=0, p=None, p1=1.0, m=None, m1=0.0,
             out=P, stream=None)
    return N.load().moc_sample_tokens(*{**d, **c}.values())


SHARED = [dict(dim=96), dict(page=24), dict(page=512), dict(code=2), dict(tokens=2), dict(tokens=-1), dict(seqs=-1),
          dict(kv_heads=0), dict(width=-1), dict(pages=-1), dict(q=None), dict(kc=None), dict(vs=None), dict(table=None),
          dict(lens=None), dict(out=None), dict(q=ctypes.c_void_p((1 << 20) + 2)), dict(q_ld=257), dict(o_lh=60),
          dict(kc=ctypes.c_void_p((1 << 20) + 8))]


@pytest.mark.parametrize("bad", SHARED, ids=str)
def test_c_entries_refuse(bad):
    for entry, name in ((_c_append, "moc_paged_append_bf16"), (_c_attention, "moc_paged_attention_bf16")):
        assert entry(**bad) == N.MOC_ERR_INVALID
        assert N.last_error().startswith(name)


def test_c_entries_refuse_their_own():
    for bad in (dict(table_dtype=2), dict(cos=None), dict(k_ld=12), dict(v=None), dict(angles=-1)):
        assert _c_append(**bad) == N.MOC_ERR_INVALID
    for bad in (dict(heads=5), dict(heads=0), dict(pages=0), dict(width=(1 << 26) + 1),
                dict(width=4000)):  # the last: no workspace
        assert _c_attention(**bad) == N.MOC_ERR_INVALID, bad
    for bad in (dict(dtype=2), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(rows=-1), dict(ld=-1), dict(x=None), dict(u=None),
                dict(out=None)):
        assert _c_sample(**bad) == N.MOC_ERR_INVALID
        assert N.last_error().startswith("moc_sample_tokens")


def test_sampling_workspace():
    lib = N.load()
    assert lib.moc_sample_tokens_workspace_size(4, 32000) == 0 == lib.moc_sample_tokens_workspace_size(0, 128256)
    need = lib.moc_sample_tokens_workspace_size(2, 128256)
    assert need > 0 and need == 2 * lib.moc_sample_tokens_workspace_size(1, 128256)
    for ws, size in ((P, need - 1), (ctypes.c_void_p((1 << 20) + 8), need)):
        assert lib.moc_sample_tokens_ws(N.MOC_F32, P, 2, 128256, 128256, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, ws,
                                        size, None) == N.MOC_ERR_INVALID
        assert "workspace of %d bytes" % need in N.last_error()


def test_c_entries_take_nothing():
    assert _c_append(tokens=0, seqs=0, q=None, k=None, v=None, table=None, lens=None, out=None) == N.MOC_OK
    assert _c_attention(tokens=0, seqs=0, q=None, table=None, lens=None, out=None) == N.MOC_OK
    assert _c_sample(rows=0, x=None, u=None, out=None) == N.MOC_OK
