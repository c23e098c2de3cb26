"""Decode of a batch over a paged 8-bit cache (moc_amd/inference/batch_decode.py)
against the decode model's own prompt forward, over its bf16 cache."""
import pytest
import torch

from moc_amd import kernels as K
from moc_amd.inference.batch_decode import BatchDecoder
from moc_amd.inference.decode_model import DecodeConfig, DecoderModel

import paged_reference as R

pytestmark = pytest.mark.gpu
BF, E4, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8


def _model(row, hidden=256, heads=4, max_seq=96):
    cfg = DecodeConfig(hidden=hidden, intermediate=704, heads=heads, layers=2, vocab=500, k=hidden // 2, max_seq=max_seq)
    m = DecoderModel(row, cfg).to("cuda", BF).init_weights(5)
    # the stream at unit scale, as in test_gpu_decode_attention.py
    m.embed.weight.data.mul_(50)
    return m


def _prompts(lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 500, (n,), generator=g).cuda() for n in lengths]


@pytest.mark.parametrize("row", ["dense", "global_moc", "moc_2_8"])
@pytest.mark.parametrize("codes,share", [(I8, 0.02), (E4, 0.04)])
@pytest.mark.parametrize("heads,page", [(4, 16), (2, 64)])
def test_prompt_and_steps_match_the_bf16_cache(row, codes, share, heads, page):
    """Logits behind ragged prompts and behind single tokens.

    A value of a block is off by at most half a step: int8 2^-7 of the block's
    largest (a scale is at most twice the least one), e4m3 2^-4 of itself; spread
    evenly over the step that is 0.016 (largest 3.5 times the rms) and 0.036 of the
    rms, in the values and, through the scores, in the probabilities, so at most
    twice that of an attention output, whose branch is about a fifth of the stream
    (2 layers, weights of 0.02 over 256): 0.01 and 0.02 of the logits, doubled for
    selections that move (1e-2 was measured for bf16 roundings alone)."""
    m = _model(row, heads=heads)
    prompts = _prompts([17, 1, 40, 64])
    d = BatchDecoder(m, 6, page=page, codes=codes)
    m.allocate_cache()
    got = [d.prompt([p[:-3] if p.numel() > 3 else p for p in prompts], room=3)]
    rest = [p[-3:] if p.numel() > 3 else torch.zeros(3, dtype=torch.int64, device="cuda") for p in prompts]
    for i in range(3):
        d.tokens[:4] = torch.stack([r[i] for r in rest])
        d.lens.add_(d.live)
        got.append(d.logits(d.forward(d.tokens))[:4])
    for b, p in enumerate(prompts):
        whole = p if p.numel() > 3 else torch.cat((p, rest[b]))
        m.reset_cache()
        want = m.forward_prompt(whole[None])[0].float()
        for i in range(4):
            ref = want[whole.numel() - 4 + i]
            assert (got[i][b].float() - ref).norm() <= 2 * share * ref.norm(), (b, i)


@pytest.mark.parametrize("row", ["dense", "global_moc"])
def test_generate_graph_equals_eager(row):
    m = _model(row)
    prompts = _prompts([5, 31, 16])
    for settings in (dict(), dict(temperature=1.2, top_k=40, top_p=0.9), dict(
            temperature=torch.tensor([0.0, 1.0, 0.7, 0.0], device="cuda"), min_p=0.01)):
        outs = [BatchDecoder(m, 4, page=16).generate(prompts, 12, generator=torch.Generator("cuda").manual_seed(1),
                                                     graph=graph, **settings) for graph in (False, True)]
        assert torch.equal(*outs) and outs[0].shape == (3, 12) and (outs[0] >= 0).all() and (outs[0] < 500).all()


def test_a_step_draws_from_its_logits_and_grows_the_sequences():
    m = _model("dense")
    d = BatchDecoder(m, 3, page=16)
    first = d.prompt(_prompts([15, 16]), room=4)
    d.tokens[:2] = first.argmax(-1)
    for i in range(4):
        u = torch.rand(3, generator=torch.Generator().manual_seed(i)).cuda()
        before = d.tokens.clone()
        d.step(u, 0.9, 50, 0.95, 0.0)
        assert d.lens.tolist() == [16 + i, 17 + i, 0] and d.tokens[2] == before[2]
        after = d.tokens.clone()
        d.tokens.copy_(before)  # the same position again: the same keys, the same logits
        logits = d.logits(d.forward(d.tokens))
        for b in range(2):
            f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
            want, near = R.sample(logits[b].float().cpu().numpy(), float(u[b]), f32(0.9), 50, f32(0.95), 0.0)
            assert int(after[b]) == want or near < 1e-9
        d.tokens.copy_(after)


def test_slots_do_not_touch_each_other():
    """A sequence alone and beside others, in other pages: the same tokens."""
    m = _model("global_moc")
    prompts = _prompts([20, 33, 8])
    # one token a forward takes other FFN kernels than several: compare at three
    alone = [BatchDecoder(m, 3, page=16).generate([p, p, p], 8) for p in prompts]
    beside = BatchDecoder(m, 3, page=16).generate(prompts, 8)
    for a, b in zip(alone, beside):
        assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])
        # prompts of other lengths run as other products: their roundings may
        # choose another token, after which the sequences differ
        assert int((a[0] == b).int().cumprod(0).sum()) >= 1


def test_a_slot_without_room_writes_nowhere():
    """Steps past the reserved pages: no page changes, the next slot's included."""
    d = BatchDecoder(_model("global_moc"), 3, page=16)
    d.prompt(_prompts([16, 16]))
    before = [[t.view(torch.uint8).clone() if t.dtype == E4 else t.clone() for t in kv] for kv in d.kv]
    u = torch.zeros(3, device="cuda")
    for _ in range(2):
        assert d.step(u).tolist() == [0, 0, 0]
    for kv, was in zip(d.kv, before):
        for t, w in zip(kv, was):
            assert torch.equal(t.view(torch.uint8) if t.dtype == E4 else t, w)
    d.reserve([40, 16, 0])  # room again: the first goes on
    d.lens.copy_(torch.tensor([16, 16, 0], dtype=torch.int32))
    d.lens.add_(d.live)
    x = d.logits(d.forward(d.tokens))
    assert torch.isfinite(x[0]).all() and torch.isnan(x[1]).any()


def test_logits_of_nan_give_a_word_of_the_vocabulary():
    m = _model("dense")
    m.lm_head.weight.data.fill_(float("nan"))
    out = BatchDecoder(m, 2, page=16).generate(_prompts([5, 9]), 4)
    assert out.shape == (2, 4) and int(out.min()) >= 0 and int(out.max()) < 500


def test_refusals():
    m = _model("dense")
    d = BatchDecoder(m, 2, page=16, pages=5)
    with pytest.raises(ValueError):
        d.prompt([])
    with pytest.raises(ValueError):
        d.prompt(_prompts([3, 3, 3]))
    with pytest.raises(ValueError):
        d.prompt([torch.empty(0, dtype=torch.int64, device="cuda")])
    with pytest.raises(ValueError, match="positions"):
        d.prompt(_prompts([90]), room=7)
    with pytest.raises(ValueError, match="pages"):
        d.prompt(_prompts([40, 40]))
    with pytest.raises(ValueError):
        d.generate(_prompts([3]), 0)
    with pytest.raises(ValueError):
        BatchDecoder(DecoderModel("dense", m.cfg), 2)
    with pytest.raises(ValueError):
        BatchDecoder(m, 0)
    d.prompt(_prompts([40, 30]))  # the pool still holds all pages
    assert d.lens.tolist() == [40, 30] and K.paged_kv(1, 1, 16, 64).k.shape == (1, 1, 16, 64)
