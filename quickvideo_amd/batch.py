"""Several sequences decoded TOGETHER over one prefilled video: beams, drafted tokens, several questions or sampled answers (the reference
hands `num_beams` and every other generation kwarg to HF generate, lvu/models/qwen25_lvu.py:744-761).

Decoding reads the whole pruned cache once per step (29 GB over 28 layers for the hour-long video); one sequence after the other, B beams
read it B times.  Here the rows of a step go through the layers as one batch:

    embed -> per layer [ add + RMSNorm -> qkv GEMM -> qp_batch_rope_append (rotation + K/V into each sequence's own pages)
                         -> qp_batch_attn (the video's rows once for all sequences, then each one's pages) -> o GEMM -> add + RMSNorm
                         -> gate|up GEMM + SwiGLU -> down GEMM ] -> RMSNorm -> lm_head

The engine's arena (video + prompt) is only read.  A sequence's own rows live in 16-row pages: forking one (beam search) shares its full
pages and copies the last, partial one; forgetting rows (refused drafts) is a smaller length."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch


class BatchDecoder:
    PAGE = 16

    @staticmethod
    def supported(eng) -> bool:
        """Engines that hold all layers and heads in one process and whose operators have the batch entry points (no pruning of the query)."""
        return (eng.tp_size == 1 and eng.pp_size == 1 and not eng.tp_on and not eng.sp_on and not eng.cfg.do_top_k_for_query and eng.D == 128
                and hasattr(eng.ops, "batch_attn"))

    def __init__(self, eng, rope_delta: int, batch: int, max_new_tokens: int, max_step: int = 1):
        """eng: prefilled (video + prompt tail).  batch sequences of up to max_new_tokens own tokens, at most max_step of them in one step."""
        if not self.supported(eng):
            raise ValueError("BatchDecoder needs a single-process engine whose operators offer batch_attn (tensor / pipeline / group-token parallel "
                             "engines and query pruning decode one sequence at a time)")
        if batch < 1 or max_new_tokens < 1 or max_step < 1:
            raise ValueError("batch, max_new_tokens and max_step must be >= 1")
        if batch * max_step > eng.n_max:
            raise ValueError(f"{batch} sequences x {max_step} tokens exceed the engine's {eng.n_max} rows a segment")
        self.eng, self.B, self.T = eng, batch, max_step
        self.prefix = list(eng.arena.len)                              # rows of every layer all sequences share
        self.pos0 = eng.seq_pos + rope_delta                           # rotary position of a sequence's first own token
        dev, dt, L, ps = eng.device, eng.dtype, len(eng.w.layers), self.PAGE
        self.width = -(-(max_new_tokens + max_step) // ps)             # pages a sequence may need (refused drafts included)
        self.n_pages = batch * (self.width + 1)                        # + 1: the copy of a forked page is made before the old one is let go
        self.pages = torch.zeros(L, 2, self.n_pages, eng.hkv, ps, eng.D, dtype=dt, device=dev)
        self.table = torch.full((batch, self.width), -1, dtype=torch.int32, device=dev)
        self.seq_len = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.owned: List[List[int]] = [[] for _ in range(batch)]       # page numbers, in order (host mirror of the table)
        self.length = [0] * batch                                      # host mirror of seq_len
        self.users = [0] * self.n_pages                                # sequences that name a page
        self.free = list(range(self.n_pages - 1, -1, -1))
        self.ws = None
        if hasattr(eng.ops, "batch_attn_workspace"):
            need = [eng.ops.batch_attn_workspace(batch, max_step, p, self.width * ps, eng.hq, eng.hkv) for p in set(self.prefix)]
            self.ws = max(need, key=lambda t: t.numel())
        self._ws_rows = {max_step: self.ws}
        self._step: Optional[List[int]] = None                         # counts of the step whose rows keep() has not been told about

    # ------------------------------------------------------------------------------------------------------------- pages
    def _upload(self):
        rows = [own + [-1] * (self.width - len(own)) for own in self.owned]
        self.table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.seq_len.copy_(torch.tensor(self.length, dtype=torch.int32))

    def _release(self, page: int):
        self.users[page] -= 1
        if self.users[page] == 0:
            self.free.append(page)

    def _reserve(self, counts: Sequence[int]) -> bool:
        """Pages for `counts[b]` more rows of every sequence; True when the table changed."""
        grown = False
        needs = [-(-(n + c) // self.PAGE) for n, c in zip(self.length, counts)]
        for b, need in enumerate(needs):                               # (before any page is taken: a refused step changes nothing)
            if need > self.width:
                raise RuntimeError(f"sequence {b} is full ({self.length[b]} of {self.width * self.PAGE} rows)")
        for b, need in enumerate(needs):
            while len(self.owned[b]) < need:
                page = self.free.pop()
                self.users[page] = 1
                self.owned[b].append(page)
                grown = True
        return grown

    def reorder(self, parents: Sequence[int]):
        """Sequence i goes on as a copy of sequence parents[i] (beam search).  Full pages are shared; the last one of a parent with several
        children is copied for all but the first of them, because each child stores into it."""
        if len(parents) != self.B or not all(0 <= p < self.B for p in parents):
            raise ValueError(f"parents {list(parents)} for {self.B} sequences")
        if self._step is not None:
            raise RuntimeError("reorder() between step() and keep(): say first how many of the step's rows stay")
        if list(parents) == list(range(self.B)):
            return
        ps = self.PAGE
        new, copies, taken = [], [], set()
        for p in parents:
            full = self.length[p] // ps
            own = self.owned[p][:full]
            for page in own:
                self.users[page] += 1
            if self.length[p] % ps:
                last = self.owned[p][full]
                if p in taken:
                    page = self.free.pop()
                    self.users[page] = 1
                    copies.append((last, page))
                    own = own + [page]
                else:
                    taken.add(p)
                    self.users[last] += 1
                    own = own + [last]
            new.append(own)
        for own in self.owned:
            for page in own:
                self._release(page)
        if copies:
            src, dst = (torch.tensor(x, dtype=torch.long, device=self.pages.device) for x in zip(*copies))
            self.pages.index_copy_(2, dst, self.pages.index_select(2, src))
        self.owned = [list(o) for o in new]
        self.length = [self.length[p] for p in parents]
        self._upload()

    # -------------------------------------------------------------------------------------------------------------- step
    def step(self, tokens: torch.Tensor, counts: Optional[Sequence[int]] = None) -> torch.Tensor:
        """tokens int64 [B, T] (T <= max_step): the next tokens of every sequence, counts[b] of them real (default T).  Their K/V rows are stored
        behind the sequence's rows; -> bf16 logits [B, T, V].  keep() then says how many stay."""
        eng, ops, s = self.eng, self.eng.ops, self.eng.spec
        B, T = tokens.shape
        if B != self.B or not 1 <= T <= self.T:
            raise ValueError(f"tokens {tuple(tokens.shape)} for {self.B} sequences of at most {self.T} tokens a step")
        counts = [T] * B if counts is None else [int(c) for c in counts]
        if len(counts) != B or not all(0 <= c <= T for c in counts):
            raise ValueError(f"counts {counts} for {B} sequences of {T} tokens")
        if self._reserve(counts):
            self._upload()
        n_new = None if counts == [T] * B else torch.tensor(counts, dtype=torch.int32, device=eng.device)
        ws = self._ws_rows.get(T, self.ws)
        if T not in self._ws_rows and self.ws is not None:             # (the launch plan, and with it the scratch, is chosen per shape)
            ws = max((ops.batch_attn_workspace(B, T, p, self.width * self.PAGE, eng.hq, eng.hkv) for p in set(self.prefix)), key=lambda t: t.numel())
            self._ws_rows[T] = ws
        n, D, hq, hkv = B * T, eng.D, eng.hq, eng.hkv
        h, x, o, dn, act = eng.b_h[:n], eng.b_x[:n], eng.b_o[:n], eng.b_dn[:n], eng.b_act[:n]
        qkv, q, att = eng.b_qkv[:n], eng.b_q[:n], eng.b_att[:n]
        h.copy_(eng.embed_tokens(tokens.reshape(-1)))
        pos = (self.seq_len.long()[:, None] + torch.arange(self.pos0, self.pos0 + T, device=eng.device)).reshape(1, n).expand(3, n).contiguous()
        cos, sin = ops.mrope_table(pos, s.mrope_section, s.rope_theta, D)
        self._step = counts
        delta = None
        for l, lw in enumerate(eng.w.layers):
            kp, vp = self.pages[l, 0], self.pages[l, 1]
            ops.add_rmsnorm(h, delta, lw.ln1, x, s.rms_eps)
            eng._linear("qkv", x, lw.w_qkv, qkv, lw.b_qkv)
            ops.batch_rope_append(qkv.view(B, T, -1), cos, sin, self.seq_len, n_new, self.table, kp, vp, hq, hkv, D, q.view(B, T, hq, D))
            ops.batch_attn(q.view(B, T, hq, D), eng.arena.k(l), eng.arena.v(l), eng.arena.head_stride, self.prefix[l], kp, vp, self.table, self.seq_len, n_new,
                           hq, hkv, D, D ** -0.5, att.view(B, T, hq, D), ws)
            eng._linear("o", att.view(n, hq * D), lw.w_o, o)
            ops.add_rmsnorm(h, o, lw.ln2, x, s.rms_eps)
            eng._gate_up_swiglu(x, lw, act)
            eng._linear("down", act, lw.w_down, dn)
            delta = dn
        ops.add_rmsnorm(h, delta, eng.w.norm, x, s.rms_eps)
        return torch.mm(x, eng.w.lm_head.t()).view(B, T, -1)

    def keep(self, counts: Sequence[int]):
        """counts[b] of the last step's tokens of sequence b stay; the rows behind them are overwritten by the next step."""
        counts = [int(c) for c in counts]
        if self._step is None or len(counts) != self.B or not all(0 <= c <= n for c, n in zip(counts, self._step)):
            raise ValueError(f"keep({counts}): the last step stored {self._step} rows")
        self._step = None
        self.length = [n + c for n, c in zip(self.length, counts)]
        self.seq_len.copy_(torch.tensor(self.length, dtype=torch.int32))


def lookup_drafts(ids: Sequence[int], k: int, max_ngram: int = 2) -> List[int]:
    """Up to k tokens that followed the latest earlier occurrence of the last max_ngram (else fewer) tokens of `ids` (HF's prompt lookup)."""
    ids = list(ids)
    for n in range(min(max_ngram, len(ids) - 1), 0, -1):
        tail = ids[-n:]
        for i in range(len(ids) - n - 1, -1, -1):
            if ids[i:i + n] == tail:
                return ids[i + n:i + n + k]
    return []


class LookupDecoder:
    """One sequence, drafted from its own context: up to `k` drafts are run through the model together with the last token (one pass over the
    cache), qp_verify_drafts keeps those that the model stands by and adds the token that follows them.  Greedy: the tokens of the plain greedy loop
    (computed by GEMMs instead of matrix-vector products, so a tie within their rounding may fall the other way).  Sampled: the same distribution."""

    def __init__(self, eng, rope_delta: int, max_new_tokens: int, k: int, selector):
        if k < 1:
            raise ValueError(f"lookup_tokens (={k}) must be >= 1")
        k = min(int(k), 255)                                           # drafts of one qp_verify_drafts call
        self.dec = BatchDecoder(eng, rope_delta, 1, max_new_tokens, max_step=k + 1)
        self.k, self.sel, self.V = k, selector, eng.w.lm_head.shape[0]
        dev = eng.device
        self.accepted = torch.zeros(1, dtype=torch.int32, device=dev)
        self.tokens = torch.zeros(1, k + 1, dtype=torch.int64, device=dev)
        self.n_draft = torch.zeros(1, dtype=torch.int32, device=dev)
        self.drafts = torch.zeros(1, k, dtype=torch.int64, device=dev)
        make = getattr(eng.ops, "verify_drafts_workspace", None)
        self.ws = make(1, k, self.V) if make else None
        self.steps = self.drafted = self.stood = 0

    def _scores(self, logits: torch.Tensor, drafts: List[int]) -> torch.Tensor:
        """What the selector would choose from, row by row: row t follows drafts[:t]."""
        sel = self.sel
        if sel.trivial:
            return logits
        seen = sel.seen
        rows = []
        for t in range(logits.shape[1]):
            if seen is not None and t and t <= len(drafts):
                sel.seen = sel.seen.clone()
                sel.seen[drafts[t - 1]] = True
            rows.append(sel.process(logits[0, t]))
        sel.seen = seen
        return torch.stack(rows)[None]

    def generate(self, first_token: int, context: Sequence[int], max_new_tokens: int, eos: Sequence[int] = ()) -> List[int]:
        """Tokens after `first_token` (which is already chosen), at most max_new_tokens of them; context: the prompt's ids."""
        dec, sel, eng = self.dec, self.sel, self.dec.eng
        dev, eos = eng.device, set(eos)
        ids, out = list(context) + [int(first_token)], []
        while len(out) < max_new_tokens and ids[-1] not in eos:
            drafts = lookup_drafts(ids, min(self.k, max_new_tokens - len(out) - 1))     # (no drafts past the last token wanted)
            step = [ids[-1]] + drafts
            tokens = torch.zeros(1, self.k + 1, dtype=torch.int64)
            tokens[0, :len(step)] = torch.tensor(step)
            logits = dec.step(tokens.to(dev), [len(step)])
            self.drafts.copy_(tokens[:, 1:])
            self.n_draft.fill_(len(drafts))
            sampled = sel.do_sample and not sel.trivial
            u = torch.rand(1, self.k + 1, generator=sel.gen, device=dev) if sampled else None
            eng.ops.verify_drafts(self._scores(logits, drafts), self.drafts, self.n_draft, None, u, 1.0 if sampled else 0.0, self.accepted, self.tokens, self.ws)
            row = self.tokens[0].tolist()                              # (the step's only host round trip)
            new = [t for t in row if t >= 0]
            if not new:
                raise RuntimeError("the model's logits offer no token")
            for i, t in enumerate(new):
                if t in eos:
                    new = new[:i + 1]
                    break
            dec.keep([len(new)])                                       # the last token and the drafts before the newest one
            self.steps, self.drafted, self.stood = self.steps + 1, self.drafted + len(drafts), self.stood + len(new) - 1
            if sel.seen is not None:
                sel.seen[torch.tensor(new, device=sel.seen.device)] = True
            ids += new
            out += new
        return out[:max_new_tokens]
