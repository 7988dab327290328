"""Host logic of quickvideo_amd/batch.py on the CPU doubles: a batch decoded together gives every sequence what it gets alone; forked sequences do not
disturb one another; refused drafts leave nothing behind; prompt lookup gives the greedy answer; batched beams the beams' answer."""
import numpy as np
import pytest
import torch

from batch_oracle import BatchOracleOps
from oracle import qp_oracle as O
from quickvideo_amd.batch import BatchDecoder, LookupDecoder, lookup_drafts
from quickvideo_amd.beam import EngineBeams, beam_search
from quickvideo_amd.engine import QuickPrefillEngine
from quickvideo_amd.lvu_config import LVUConfig
from quickvideo_amd.sampling import TokenSelector
from quickvideo_amd.spec import TextSpec
from quickvideo_amd.weights import DecoderWeights

DIMS = dict(hidden=256, n_heads=2, n_kv_heads=1, head_dim=128, intermediate=256, n_layers=2, vocab=64)


def near(got, ref):
    """Two bf16 steps (2^-7) of the largest logit: the two results are each rounded by up to half a step, and the hidden rows behind them differ by single
    bf16 steps (keys rounded once instead of three times, other orders of summation), which a 256-term product averages to less than one step."""
    return (got.float() - ref).abs().max().item() <= 2 * 2.0 ** -7 * ref.abs().max().item()


def engine(seed=13, lm=8.0, **cfg):
    so, spec = O.TextSpec(**DIMS), TextSpec(**DIMS)
    w = {k: (v * (lm if "lm_head" in k else 1.0)).to(torch.bfloat16) for k, v in O.synthetic_text_weights(so, seed=seed, norm_jitter=0.1).items()}
    rs = np.random.RandomState(3)
    groups, tail = [20, 24], 6
    T = sum(groups) + tail
    embeds = torch.from_numpy(rs.standard_normal((T, 256)).astype(np.float32) * 0.5).to(torch.bfloat16)
    pos = torch.from_numpy(np.tile(np.arange(T, dtype=np.int64), (3, 1)))
    eng = QuickPrefillEngine(DecoderWeights.from_named(spec, w, "cpu"), LVUConfig("x", top_p=0.5, video_group_size=4, **cfg), capacity=T + 64, max_group_tokens=64,
                             device="cpu", ops=BatchOracleOps())
    st = 0
    for n in groups:
        eng.prefill_group(embeds[st:st + n], pos[:, st:st + n]); st += n
    return eng, eng.prefill_tail(embeds[st:], pos[:, st:])


def alone(eng, tokens):
    """fp32 logits after each token of ONE sequence by the engine's own decode step; the engine is left as it was."""
    lens, at = list(eng.arena.len), eng.seq_pos
    out = [eng.decode_step(eng.embed_tokens(torch.tensor([t])), 0) for t in tokens]
    eng.arena.len, eng.seq_pos = lens, at
    return torch.stack(out)


def test_batch_steps_equal_sequences_alone():
    eng, _ = engine()
    seqs = [[5, 9, 11, 60, 2, 3, 3, 8, 1, 44, 7, 7, 7, 12, 30, 31, 32, 33, 34, 35], [1], [40, 41, 42, 43, 44]]
    dec = BatchDecoder(eng, 0, 3, 24, max_step=6)
    got = [[] for _ in seqs]
    at = [0, 0, 0]
    shared = [eng.arena.buf[l, :, :, :n].clone() for l, n in enumerate(eng.arena.len)]
    while any(a < len(s) for a, s in zip(at, seqs)):
        counts = [min(6 - 2 * b, len(s) - a) for b, (a, s) in enumerate(zip(at, seqs))]
        tokens = torch.zeros(3, 6, dtype=torch.int64)
        for b, c in enumerate(counts):
            tokens[b, :c] = torch.tensor(seqs[b][at[b]:at[b] + c])
        logits = dec.step(tokens, counts)
        dec.keep(counts)
        for b, c in enumerate(counts):
            got[b] += list(logits[b, :c].float())
            at[b] += c
    assert all(torch.equal(eng.arena.buf[l, :, :, :n], shared[l]) for l, n in enumerate(eng.arena.len)) and dec.length == [len(s) for s in seqs]
    for b, s in enumerate(seqs):
        assert near(torch.stack(got[b]), alone(eng, s))


def test_forks_share_full_pages_and_do_not_disturb_each_other():
    eng, _ = engine()
    rs = np.random.RandomState(1)
    dec = BatchDecoder(eng, 0, 4, 40)
    seqs = [[] for _ in range(4)]
    for step in range(38):
        if step % 3 == 2 or step in (16, 17):
            parents = rs.randint(0, 4, 4).tolist()
            dec.reorder(parents)
            seqs = [list(seqs[p]) for p in parents]
        toks = rs.randint(0, 64, 4).tolist()
        logits = dec.step(torch.tensor(toks)[:, None])
        dec.keep([1] * 4)
        seqs = [s + [t] for s, t in zip(seqs, toks)]
        used = sorted(p for own in dec.owned for p in own)
        assert all(dec.users[p] == used.count(p) for p in set(used)) and sorted(dec.free + list(set(used))) == list(range(dec.n_pages))
        last = [own[-1] for own in dec.owned]
        assert len(set(last)) == 4 or dec.length[0] % dec.PAGE == 0            # a page that will be stored into has one owner
        if step in (5, 17, 37):
            for b in range(4):
                assert near(logits[b, 0], alone(eng, seqs[b])[-1])
    with pytest.raises(ValueError, match="parents"):
        dec.reorder([0, 1, 2, 4])
    with pytest.raises(ValueError, match="parents"):
        dec.reorder([0, 1, 2])


def test_refused_tokens_are_forgotten():
    eng, _ = engine()
    dec = BatchDecoder(eng, 0, 2, 40, max_step=20)
    dec.step(torch.randint(0, 64, (2, 20), generator=torch.Generator().manual_seed(1)), [20, 18])
    dec.keep([0, 1])
    assert dec.length == [0, 1]
    first = dec.step(torch.tensor([[7, 8, 9], [50, 51, 52]]), [3, 3])
    dec.keep([3, 3])
    assert near(first[0], alone(eng, [7, 8, 9]))


def test_batch_decoder_refusals():
    eng, _ = engine()
    for args, word in (((0, 4), "batch"), ((2, 0), "max_new_tokens"), ((2, 4, 0), "max_step"), ((40, 4, 2), "rows")):
        with pytest.raises(ValueError, match=word):
            BatchDecoder(eng, 0, *args)
    dec = BatchDecoder(eng, 0, 2, 20, max_step=2)
    for bad in (torch.zeros(3, 1, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tokens"):
            dec.step(bad)
    with pytest.raises(ValueError, match="counts"):
        dec.step(torch.zeros(2, 2, dtype=torch.int64), [3, 0])
    for _ in range(16):
        dec.step(torch.zeros(2, 2, dtype=torch.int64)); dec.keep([2, 2])
    with pytest.raises(RuntimeError, match="full"):
        dec.step(torch.zeros(2, 2, dtype=torch.int64))
    query, _ = engine()
    query.cfg.do_top_k_for_query = True
    assert not BatchDecoder.supported(query)
    with pytest.raises(ValueError, match="single-process"):
        BatchDecoder(query, 0, 1, 4)


@pytest.mark.parametrize("ids,k,want", [([1, 2, 3, 1, 2], 3, [3, 1, 2]), ([1, 2, 3, 1, 2], 1, [3]), ([5, 9, 5], 4, [9, 5]), ([1, 2, 3], 4, []), ([1], 3, []), ([], 3, []),
                                        ([4, 4, 4], 2, [4]), ([7, 8, 1, 7, 8, 2, 7, 8], 2, [2, 7]), ([1, 2, 1], 0, [])])
def test_lookup_drafts(ids, k, want):
    assert lookup_drafts(ids, k) == want


@pytest.mark.parametrize("k", [1, 3, 7])
@pytest.mark.parametrize("penalty", [1.0, 1.3])
def test_lookup_gives_the_greedy_answer(k, penalty):
    for seed in (13, 14, 15):
        eng, first = engine(seed)
        tok = int(first.argmax())
        context = [3, 9, tok, 5, 3, 9]
        ref, sel = [], TokenSelector(repetition_penalty=penalty)
        sel.observe(context, 64, "cpu")
        if sel.seen is not None:
            sel.seen[tok] = True
        lens, at, t = list(eng.arena.len), eng.seq_pos, tok
        for _ in range(20):
            t = sel.select(eng.decode_step(eng.embed_tokens(torch.tensor([t])), 0))
            ref.append(t)
        eng.arena.len, eng.seq_pos = lens, at
        sel = TokenSelector(repetition_penalty=penalty)
        sel.observe(context, 64, "cpu")
        if sel.seen is not None:
            sel.seen[tok] = True
        look = LookupDecoder(eng, 0, 20, k, sel)
        assert look.generate(tok, context, 20) == ref
        if ref[4] in ref[:4]:
            eos = ref[4]
            look = LookupDecoder(eng, 0, 20, k, TokenSelector(repetition_penalty=1.0))
            if penalty == 1.0:
                assert look.generate(tok, context, 20, [eos]) == ref[:ref.index(eos) + 1]


def test_lookup_saves_steps_on_a_repeating_answer():
    eng, first = engine(13)
    tok = int(first.argmax())
    plain = LookupDecoder(eng, 0, 40, 1, TokenSelector())
    out = plain.generate(tok, [], 40)
    long = LookupDecoder(eng, 0, 40, 7, TokenSelector())
    assert long.generate(tok, [tok] + out, 40) == out and long.stood > 0 and long.steps + long.stood >= 40 and long.steps < 40


def test_lookup_sampling_runs_and_stops():
    eng, first = engine(13)
    sel = TokenSelector(do_sample=True, temperature=0.8, top_k=12, top_p=0.9, seed=5)
    out = LookupDecoder(eng, 0, 12, 4, sel).generate(int(first.argmax()), [1, 2, 3], 12)
    assert len(out) == 12 and all(0 <= t < 64 for t in out)
    with pytest.raises(ValueError, match="lookup_tokens"):
        LookupDecoder(eng, 0, 12, 0, sel)


@pytest.mark.parametrize("B,mnt", [(3, 5), (4, 20)])
def test_batched_beams_give_the_beams_answer(B, mnt):
    eng, first = engine()
    a = EngineBeams(eng, 0, B, mnt)
    want = beam_search(first, a.advance, B, mnt, eos_ids=(7,))
    a.finish(len(want))
    b = EngineBeams(eng, 0, B, mnt, batched=True)
    got = beam_search(first, b.advance, B, mnt, eos_ids=(7,))
    b.finish(len(got))
    assert got == want


def test_generate_through_the_public_interface():
    """LVU.generate: `batched_beams` and `lookup_tokens` give what the call without them gives; they are refused where they cannot work."""
    import lvu
    from quickvideo_amd.lvu import load_native_model
    obj = lvu.LVU(lvu.LVUConfig("synthetic:tiny", top_p=0.5, video_group_size=4, num_frames=8), model=load_native_model("synthetic:tiny", device="cpu"))
    obj._ops = BatchOracleOps()
    video = "synthetic://?frames=16&h=56&w=84&fps=2&seed=3"
    run = lambda **kw: obj.generate("What happens?", video, max_new_tokens=6, eos_token_id=None, **kw)[0]                    # noqa: E731
    greedy = run()
    assert run(lookup_tokens=3) == greedy and run(lookup_tokens=1) == greedy and run(lookup_tokens=3, repetition_penalty=1.2) == run(repetition_penalty=1.2)
    assert run(num_beams=3, batched_beams=True) == run(num_beams=3)
    assert run(num_beams=3, batched_beams=True, do_sample=True, seed=4) == run(num_beams=3, batched_beams=True, do_sample=True, seed=4)
    a = run(lookup_tokens=2, do_sample=True, temperature=5.0, seed=7)
    assert a == run(lookup_tokens=2, do_sample=True, temperature=5.0, seed=7) and a.count("<tok_") == 6
    assert run() == greedy                                                   # nothing of the above stays behind
    for kw, word in ((dict(lookup_tokens=2, num_beams=2), "one beam"), (dict(lookup_tokens=-1), ">= 1")):
        with pytest.raises(ValueError, match=word):
            run(**kw)
    obj.config.do_top_k_for_query = True
    with pytest.raises(ValueError, match="do_top_k_for_query"):
        run(num_beams=2, batched_beams=True)


def test_keep_and_reorder_refuse_what_the_last_step_did_not_store():
    eng, _ = engine()
    dec = BatchDecoder(eng, 0, 2, 40, max_step=3)
    with pytest.raises(ValueError, match="keep"):
        dec.keep([0, 0])                                               # no step yet
    dec.step(torch.tensor([[1, 2, 3], [4, 5, 6]]), [3, 1])
    with pytest.raises(RuntimeError, match="keep"):
        dec.reorder([1, 0])
    for bad in ([3, 2], [-1, 1], [3], [3, 1, 0]):
        with pytest.raises(ValueError, match="keep"):
            dec.keep(bad)
    dec.keep([3, 1])
    assert dec.length == [3, 1]
    with pytest.raises(ValueError, match="keep"):
        dec.keep([1, 1])                                               # the same step twice
    dec.reorder([1, 0])
    assert dec.length == [1, 3]


def test_a_refused_step_changes_nothing():
    """Sequence 1 is full, sequence 0 needs a new page: the step is refused before a page is taken, and sequence 0 goes on alone."""
    eng, _ = engine()
    dec = BatchDecoder(eng, 0, 2, 31, max_step=1)
    seq = []
    for i in range(32):
        dec.step(torch.tensor([[i % 7], [i % 5]]), [int(i < 16), 1])
        dec.keep([int(i < 16), 1])
        if i < 16:
            seq.append(i % 7)
    assert dec.length == [16, 32]
    owned = [list(o) for o in dec.owned]
    with pytest.raises(RuntimeError, match="full"):
        dec.step(torch.tensor([[9], [9]]))
    assert dec.owned == owned
    logits = dec.step(torch.tensor([[9], [0]]), [1, 0])
    dec.keep([1, 0])
    assert near(logits[0], alone(eng, seq + [9])[-1:])


def test_batched_beams_with_one_beam_is_the_call_without_it():
    import lvu
    from quickvideo_amd.lvu import load_native_model
    obj = lvu.LVU(lvu.LVUConfig("synthetic:tiny", top_p=0.5, video_group_size=4, num_frames=8), model=load_native_model("synthetic:tiny", device="cpu"))
    obj._ops = BatchOracleOps()
    run = lambda **kw: obj.generate("What happens?", "synthetic://?frames=16&h=56&w=84&fps=2&seed=3", max_new_tokens=6, eos_token_id=None, **kw)[0]      # noqa: E731
    assert run(num_beams=1, batched_beams=True) == run(batched_beams=True) == run()
    assert run(batched_beams=True, lookup_tokens=2) == run()
