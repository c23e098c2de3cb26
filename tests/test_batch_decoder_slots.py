"""BatchDecoder's slots (moc_amd/inference/batch_decode.py) over plain operators on
the CPU: what is stored where, and that a sequence which waits goes on as one that
did not."""
import math

import pytest
import torch

from moc_amd import kernels as K
from moc_amd.inference.batch_decode import BatchDecoder
from moc_amd.inference.decode_model import DecodeConfig, DecoderModel

import paged_reference as R

PAGE, VOCAB = 16, 50


class _Cache:
    """Keys and values of a pool, any value exactly; places start as another
    sequence's."""

    def __init__(self, pages, heads, dim, seed):
        g = torch.Generator().manual_seed(seed)
        self.k, self.v = (3 * torch.randn(pages, heads, PAGE, dim, generator=g) for _ in range(2))


def _append(q, k, v, cos, sin, kv, table, lens, cu=None):
    turned = [R.rotated(x, cos, sin, lens, cu).float() for x in (q, k)]
    for b, start, n, length in R.spans(q.shape[0], lens, cu):
        for i in range(n):
            pos = length - n + i
            page = int(table[b, pos // PAGE]) if 0 <= pos < table.shape[1] * PAGE else -1
            if page >= 0:
                kv.k[page, :, pos % PAGE], kv.v[page, :, pos % PAGE] = turned[1][start + i], v[start + i].float()
    return turned[0].to(q.dtype)


def _attention(q, kv, table, lens, cu=None, *, scale=None):
    o = torch.zeros_like(q)
    for b, start, n, length in R.spans(q.shape[0], lens, cu):
        for i in range(n):
            sees = length - n + i + 1
            if sees <= 0:
                continue
            at = [int(table[b, p // PAGE]) if p < table.shape[1] * PAGE else -1 for p in range(sees)]
            if min(at) < 0:
                o[start + i] = math.nan
                continue
            k, v = (torch.stack([c[j, :, p % PAGE] for p, j in enumerate(at)], 1) for c in (kv.k, kv.v))
            p = torch.softmax(scale * (k @ q[start + i].float()[..., None]), 1)
            o[start + i] = (p * v).sum(1).to(o.dtype)
    return o


def _sample(logits, u, *settings):
    best = logits.float().nan_to_num(nan=-math.inf).argmax(-1)
    return torch.where(logits.isnan().all(-1), -1, best)


@pytest.fixture
def decoder(monkeypatch):
    """A maker of decoders of one small model over caches of stale contents."""
    monkeypatch.setattr(K, "paged_append", _append)
    monkeypatch.setattr(K, "paged_attention", _attention)
    monkeypatch.setattr(K, "sample_tokens", _sample)
    cfg = DecodeConfig(hidden=128, intermediate=96, heads=2, layers=2, vocab=VOCAB, k=48, max_seq=72)
    model = DecoderModel("dense", cfg).to(torch.bfloat16).init_weights(2)
    model.embed.weight.data.mul_(50)

    def make(slots, pages=None):
        d = BatchDecoder(model, slots, page=PAGE, pages=pages)
        d.kv = [_Cache(d.pages, cfg.heads, cfg.hidden // cfg.heads, seed) for seed in range(cfg.layers)]
        return d

    return make


def _prompts(lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g) for n in lengths]


def _begin(d, lengths, room):
    d.tokens[:len(lengths)] = d.prompt(_prompts(lengths), room=room).argmax(-1)
    return d


def _cached(d, slot):
    """Keys and values of a slot's positions, all layers."""
    at = [(int(d.table[slot, p // PAGE]), p % PAGE) for p in range(int(d.lens[slot]))]
    return torch.stack([torch.stack([c[j, :, p] for j, p in at]) for kv in d.kv for c in (kv.k, kv.v)])


def _steps(d, n):
    return [d.step(torch.zeros(d.slots)).clone() for _ in range(n)]


def test_a_slot_out_of_use_is_left_alone(decoder):
    """reserve(0) for some steps: nothing of the slot changes, and back in use it
    goes on as if there had been no pause."""
    whole = _begin(decoder(3), [17, 15, 30], room=12)
    want = torch.stack(_steps(whole, 9))
    d = _begin(decoder(3), [17, 15, 30], room=12)
    _steps(d, 2)
    before, pending = _cached(d, 0), int(d.tokens[0])
    d.reserve([0, 27, 42])
    for _ in range(3):
        assert int(d.step(torch.zeros(3))[0]) == pending
    assert d.lens.tolist() == [19, 20, 35] and torch.equal(_cached(d, 0), before)
    d.reserve([29, 27, 42])
    rest = torch.stack(_steps(d, 7))
    assert torch.equal(rest[:, 0], want[2:, 0]) and torch.equal(rest[:4, 1:], want[5:, 1:])
    assert torch.equal(_cached(d, 0), _cached(whole, 0))


def test_a_full_slot_waits_for_room(decoder):
    """Steps past the pages that it holds leave its length and its pending token;
    with room again it goes on as if it had had it from the start."""
    whole = _begin(decoder(2), [16, 3], room=9)
    want = torch.stack(_steps(whole, 8))
    d = _begin(decoder(2), [16, 3], room=0)
    pending = d.tokens.clone()
    first = torch.stack(_steps(d, 3))
    assert d.lens.tolist() == [16, 6] and (first[:, 0] == pending[0]).all()
    assert torch.equal(first[:, 1], want[:3, 1])
    d.reserve([40, 40])
    rest = torch.stack(_steps(d, 8))
    assert d.lens.tolist() == [24, 14]
    assert torch.equal(rest[:, 0], want[:, 0]) and torch.equal(rest[:5, 1], want[3:, 1])
    assert torch.equal(_cached(d, 0), _cached(whole, 0))


def test_a_slot_stops_at_the_models_last_position(decoder):
    """72 positions in pages of 16: the last page has places that no angle has."""
    d = _begin(decoder(1), [70], room=2)
    _steps(d, 4)
    assert d.lens.tolist() == [72]


def test_a_capture_that_fails_changes_nothing(decoder, monkeypatch):
    """The sequences go on after it, as if it had not been tried."""
    whole = _begin(decoder(2), [5, 9], room=5)
    want = torch.stack(_steps(whole, 4))
    d = _begin(decoder(2), [5, 9], room=5)

    def fails(*a):
        raise RuntimeError("no capture")

    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "device", fails)
        with pytest.raises(RuntimeError, match="no capture"):
            d._capture(torch.zeros(2), (0.0, 0, 1.0, 0.0))
    assert d.lens.tolist() == [5, 9] and d.live.tolist() == [1, 1]
    assert torch.equal(torch.stack(_steps(d, 4)), want)


def test_a_refused_prompt_leaves_the_running_slots(decoder):
    """Too long, too many pages, none, room below 0: the sequences go on."""
    whole = _begin(decoder(2, pages=5), [5, 9], room=5)
    want = torch.stack(_steps(whole, 4))
    d = _begin(decoder(2, pages=5), [5, 9], room=5)
    for prompts, room in ((_prompts([70]), 3), (_prompts([40, 40]), 0), ([], 0), (_prompts([4, 4]), -1),
                          (_prompts([4, 0]), 0)):
        with pytest.raises(ValueError):
            d.prompt(prompts, room=room)
    assert torch.equal(torch.stack(_steps(d, 4)), want)
    assert d.prompt(_prompts([40, 40 - PAGE]), room=0).shape == (2, VOCAB)  # all pages


def test_what_was_drawn_is_told_from_what_was_not(decoder):
    """drawn: the id; -1 behind logits of NaN, whose slot gets token 0; -2 where no
    step was taken, whose slot keeps its token."""
    d = _begin(decoder(4), [16, 5, 9], room=0)
    assert d.drawn.tolist() == [-2] * 4
    d.tokens[2] = VOCAB - 1
    d.model.embed.weight.data[VOCAB - 1] = math.nan
    d.reserve([16, 8, 12, 0])
    before = d.tokens.clone()
    after = d.step(torch.zeros(4))
    assert d.drawn.tolist() == [-2, int(after[1]), -1, -2]
    assert after[0] == before[0] and after[2] == 0 and after[3] == before[3]
    d.prompt(_prompts([3]))
    assert d.drawn.tolist() == [-2] * 4


def test_a_refused_step_is_no_step(decoder, monkeypatch):
    """Settings that the draw refuses: the next step stores the same tokens at the
    same positions."""
    whole = _begin(decoder(2), [5, 15], room=6)
    want = torch.stack(_steps(whole, 5))
    d = _begin(decoder(2), [5, 15], room=6)
    _steps(d, 1)

    def refuses(*a):
        raise ValueError("settings")

    for _ in range(2):
        with monkeypatch.context() as m:
            m.setattr(K, "sample_tokens", refuses)
            with pytest.raises(ValueError, match="settings"):
                d.step(torch.zeros(2))
        assert d.lens.tolist() == [6, 16]
    assert torch.equal(torch.stack(_steps(d, 4)), want[1:])
    assert all(torch.equal(_cached(d, b), _cached(whole, b)) for b in range(2))
