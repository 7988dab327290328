"""The batch operators together, as a user runs them: BatchDecoder / LookupDecoder / batched beams on the HIP library against the engine's own
one-sequence decode."""
import numpy as np
import pytest
import torch

from oracle import qp_oracle as O
from quickvideo_amd.batch import BatchDecoder, LookupDecoder
from quickvideo_amd.beam import EngineBeams, beam_search
from quickvideo_amd.engine import QuickPrefillEngine
from quickvideo_amd.lvu_config import LVUConfig
from quickvideo_amd.sampling import TokenSelector
from quickvideo_amd.spec import TextSpec
from quickvideo_amd.weights import DecoderWeights

pytestmark = pytest.mark.gpu


def engine(heads=(7, 1), groups=(320, 256, 384), vocab=512, seed=5, lm=4.0):
    hq, hkv = heads
    dims = dict(hidden=512, n_heads=hq, n_kv_heads=hkv, head_dim=128, intermediate=768, n_layers=2, vocab=vocab)
    w = {k: (v * (lm if "lm_head" in k else 1.0)).to(torch.bfloat16) for k, v in O.synthetic_text_weights(O.TextSpec(**dims), seed=seed, norm_jitter=0.1).items()}
    spec, tail = TextSpec(**dims), 21
    T = sum(groups) + tail
    rs = np.random.RandomState(seed)
    e = torch.from_numpy(rs.standard_normal((T, 512)).astype(np.float32) * 0.5).to(torch.bfloat16).cuda()
    pos = torch.from_numpy(np.tile(np.arange(T, dtype=np.int64), (3, 1))).cuda()
    eng = QuickPrefillEngine(DecoderWeights.from_named(spec, w, "cuda:0"), LVUConfig("x", top_p=0.5, video_group_size=4), capacity=T + 128, max_group_tokens=max(groups),
                             device="cuda:0")
    st = 0
    for n in groups:
        eng.prefill_group(e[st:st + n], pos[:, st:st + n]); st += n
    return eng, eng.prefill_tail(e[st:], pos[:, st:])


def alone(eng, tokens):
    lens, at = list(eng.arena.len), eng.seq_pos
    out = [eng.decode_step(eng.embed_tokens(torch.tensor([t])), 0).float().cpu() for t in tokens]
    eng.arena.len, eng.seq_pos = lens, at
    return torch.stack(out)


def near(got, ref):
    """Two bf16 steps (2^-7) of the largest logit, as in the CPU test of the same decoder: two final roundings, and hidden rows that differ by single steps."""
    d = (got.float().cpu() - ref).abs().max().item()
    assert d <= 2 * 2.0 ** -7 * ref.abs().max().item(), (d, ref.abs().max().item())


@pytest.mark.parametrize("heads", [(7, 1), (8, 2), (4, 4)])
def test_batch_decoder_equals_sequences_alone(heads):
    eng, _ = engine(heads)
    seqs = [[5, 9, 11, 60, 2, 3, 3, 8, 1, 44, 7, 7, 7, 12, 30, 31, 32, 33, 34, 35, 100, 200, 300, 400], [1], [40, 41, 42, 43, 44]]
    dec = BatchDecoder(eng, 0, 3, 40, max_step=9)
    shared = [eng.arena.buf[l, :, :, :n].clone() for l, n in enumerate(eng.arena.len)]
    got, at = [[] for _ in seqs], [0, 0, 0]
    while any(a < len(s) for a, s in zip(at, seqs)):
        counts = [min(9 - 3 * b, len(s) - a) for b, (a, s) in enumerate(zip(at, seqs))]
        tokens = torch.zeros(3, 9, dtype=torch.int64, device="cuda")
        for b, c in enumerate(counts):
            tokens[b, :c] = torch.tensor(seqs[b][at[b]:at[b] + c])
        logits = dec.step(tokens, counts)
        dec.keep(counts)
        for b, c in enumerate(counts):
            got[b] += list(logits[b, :c].float().cpu())
            at[b] += c
    assert all(torch.equal(eng.arena.buf[l, :, :, :n], shared[l]) for l, n in enumerate(eng.arena.len))
    for b, s in enumerate(seqs):
        near(torch.stack(got[b]), alone(eng, s))


def test_forked_sequences_on_the_gpu():
    eng, _ = engine()
    rs = np.random.RandomState(2)
    dec, seqs = BatchDecoder(eng, 0, 4, 40), [[] for _ in range(4)]
    for step in range(36):
        if step % 4 == 3 or step == 16:
            parents = rs.randint(0, 4, 4).tolist()
            dec.reorder(parents)
            seqs = [list(seqs[p]) for p in parents]
        toks = rs.randint(0, 512, 4).tolist()
        logits = dec.step(torch.tensor(toks, device="cuda")[:, None])
        dec.keep([1] * 4)
        seqs = [s + [t] for s, t in zip(seqs, toks)]
    for b in range(4):
        near(logits[b, 0], alone(eng, seqs[b])[-1])


def test_batched_beams_follow_the_sequential_ones():
    """Scores of the batched search's answer, computed by the sequential decode, are as good as the sequential search's answer (ties within the rounding
    of the logits may fall either way): the two accumulated log-probabilities differ by at most one logit rounding (2 * 2^-8 of the largest) a token."""
    eng, first = engine()
    B, mnt = 4, 12

    def score(ans):
        rows = torch.cat([first.float().cpu()[None], alone(eng, ans[:-1])])
        return torch.log_softmax(rows, -1).gather(1, torch.tensor(ans)[:, None]).sum().item(), rows.abs().max().item()

    a = EngineBeams(eng, 0, B, mnt)
    want = beam_search(first, a.advance, B, mnt)
    a.finish(len(want))
    b = EngineBeams(eng, 0, B, mnt, batched=True)
    got = beam_search(first, b.advance, B, mnt)
    b.finish(len(got))
    (sw, top), (sg, _) = score(want), score(got)
    assert got == want or sg >= sw - mnt * 2 * 2.0 ** -8 * top, (sg, sw)


@pytest.mark.parametrize("k", [1, 5])
def test_lookup_follows_the_greedy_loop(k):
    """Every token the lookup decoder gives is the greedy one, or one whose logit is within the two paths' rounding (2 bf16 steps) of the best."""
    eng, first = engine()
    tok = int(first.argmax())
    context = [tok, 3, 9, tok]
    look = LookupDecoder(eng, 0, 30, k, TokenSelector())
    out = look.generate(tok, context, 30)
    assert len(out) == 30
    rows = alone(eng, [tok] + out[:-1])
    best = rows.max(-1).values
    taken = rows.gather(1, torch.tensor(out)[:, None])[:, 0]
    assert (best - taken <= 2 * 2 * 2.0 ** -7 * rows.abs().max()).all()
    sampled = LookupDecoder(eng, 0, 30, k, TokenSelector(do_sample=True, temperature=0.9, top_k=20, seed=3, device="cuda")).generate(tok, context, 30)
    assert len(sampled) == 30 and all(0 <= t < 512 for t in sampled)


def test_generate_on_the_gpu():
    import lvu
    from quickvideo_amd.lvu import load_native_model
    obj = lvu.LVU(lvu.LVUConfig("synthetic:tiny", top_p=0.5, video_group_size=4, num_frames=8), model=load_native_model("synthetic:tiny", device="cuda:0"))
    run = lambda **kw: obj.generate("What happens?", "synthetic://?frames=16&h=56&w=84&fps=2&seed=3", max_new_tokens=6, eos_token_id=None, **kw)[0]       # noqa: E731
    greedy = run()
    for kw in (dict(lookup_tokens=3), dict(lookup_tokens=2, do_sample=True, temperature=2.0, seed=1), dict(num_beams=3, batched_beams=True),
               dict(num_beams=3, batched_beams=True, do_sample=True, seed=2)):
        assert run(**kw).count("<tok_") >= 1
    assert run() == greedy
