"""Sizes, inputs and plain forms of the operators that decode a batch of sequences over one prefilled video:

  append   qkv rows of the batch's new tokens -> rotated queries, and keys / values stored into each sequence's own pages
  attn     attention of the batch over (the video's keys, shared by all sequences; each sequence's own paged keys)
  verify   how many drafted tokens of each sequence stand against the model's logits, and the token that follows them

`own` chooses between the plain form (elementary torch operations, the default) and the package's HIP kernels."""
import math
import random

import numpy as np
import torch

own = False
D = 128
_OPS = None


def _ops():
    global _OPS
    if _OPS is None:
        from quickvideo_amd.native import QuickPrefillOps
        _OPS = QuickPrefillOps(torch.device("cuda", torch.cuda.current_device()))
    return _OPS


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    """hq / hkv: query and key heads; batch: sequences; tokens: new tokens a sequence may have in this step (`ragged`: some have fewer);
    prefix: keys of the video that all share; suffix: about how many keys a sequence has of its own; page: rows of a page."""
    return [
        # one greedy token of a single answer: the smallest call there is, nothing but latency
        dict(name="append_token", op="append", hq=28, hkv=4, batch=1, tokens=1, suffix=11, page=16, ragged=False, shape=1),
        # one step of 16 beams of different lengths
        dict(name="append_beams", op="append", hq=28, hkv=4, batch=16, tokens=1, suffix=130, page=16, ragged=False, shape=2),
        # eight questions about one video, each appended whole (ragged, pages that end inside a question), wide model
        dict(name="append_questions", op="append", hq=64, hkv=8, batch=8, tokens=96, suffix=40, page=24, ragged=True, shape=3),
        # a short clip, one answer, one token
        dict(name="attn_clip", op="attn", hq=12, hkv=2, batch=1, tokens=1, prefix=417, suffix=9, page=16, ragged=False, shape=4),
        # four beams over a 64-frame video pruned to half
        dict(name="attn_beams", op="attn", hq=28, hkv=4, batch=4, tokens=1, prefix=11535, suffix=60, page=16, ragged=False, shape=5),
        # three answers of the wide model, up to six drafted tokens each, ragged
        dict(name="attn_drafts", op="attn", hq=64, hkv=8, batch=3, tokens=6, prefix=30737, suffix=250, page=32, ragged=True, shape=6),
        # eight beams over the hour-long video: one layer's step reads 1 GB of keys and values
        dict(name="attn_hour", op="attn", hq=28, hkv=4, batch=8, tokens=1, prefix=504015, suffix=200, page=16, ragged=False, shape=7),
        # four questions of about 60 tokens, prefilled together over a ten-minute video: matrix work, not bandwidth
        dict(name="attn_questions", op="attn", hq=28, hkv=4, batch=4, tokens=61, prefix=32785, suffix=5, page=16, ragged=True, shape=8),
        # one answer with prompt-lookup drafts (certain drafts: no probabilities of their own), sampled
        dict(name="verify_lookup", op="verify", batch=1, tokens=3, vocab=151936, dtype="bf16", probs=False, temperature=1.0, ragged=False, shape=9),
        # four answers with lookup drafts, greedy
        dict(name="verify_greedy", op="verify", batch=4, tokens=5, vocab=152064, dtype="bf16", probs=False, temperature=0.0, ragged=True, shape=10),
        # 32 answers against a draft model's probabilities, processed fp32 scores
        dict(name="verify_batch", op="verify", batch=32, tokens=4, vocab=152064, dtype="fp32", probs=True, temperature=0.7, ragged=True, shape=11),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "verify"])
    hq, hkv = rng.choice([(12, 2), (28, 4), (64, 8), (8, 1), (7, 7), (32, 2)])
    case = dict(op=op, ragged=rng.random() < 0.6, shape=rng.randrange(1 << 30))
    if op == "append":
        tokens = _log_int(rng, 1, 128)
        case.update(hq=hq, hkv=hkv, batch=_log_int(rng, 1, max(1, min(48, 700 // tokens))), tokens=tokens, suffix=_log_int(rng, 1, 200), page=rng.choice([1, 5, 16, 24, 32, 64, 128]))
    elif op == "attn":
        prefix = 0 if rng.random() < 0.08 else _log_int(rng, 1, 2_000_000 // hkv if hkv >= 4 else 504_000)
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 1, 64)
        rows = max(1, 105_000_000 // (hkv * (prefix + 1500)) // (hq // hkv))            # sequences x tokens that stay below the largest listed case
        tokens = min(tokens, rows)
        batch = _log_int(rng, 1, max(1, min(48, rows // tokens, 1024 // tokens)))
        case.update(hq=hq, hkv=hkv, batch=batch, tokens=tokens, prefix=prefix, suffix=_log_int(rng, 1, 1200 if batch <= 8 else 300), page=rng.choice([1, 7, 16, 24, 32, 64, 128]))
    else:
        vocab = _log_int(rng, 2, 152064)
        case.update(batch=_log_int(rng, 1, 32), tokens=rng.randint(0, 4), vocab=vocab, dtype=rng.choice(["bf16", "fp32"]),
                    probs=rng.random() < 0.5, temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.6]))
    return case


def _lengths(case):
    """(seq_len, n_new) of the sequences, from the case alone: keys stored before this step, new tokens of this step."""
    rng = random.Random(case["shape"])
    B, T = case["batch"], case["tokens"]
    seq = [rng.randint(case["suffix"] // 2, case["suffix"] * 3 // 2) for _ in range(B)]
    new = [rng.randint(0 if T > 1 and B > 1 else 1, T) if case["ragged"] else T for _ in range(B)]
    if B > 2:
        seq[rng.randrange(B)] = 0                                    # an answer that has just begun
    return seq, new


def _drafts(case):
    """n_draft of the sequences; -1 = an idle place of a padded batch."""
    rng = random.Random(case["shape"])
    B, T = case["batch"], case["tokens"]
    n = [rng.randint(0, T) if case["ragged"] else T for _ in range(B)]
    if case["ragged"] and B > 2:
        n[rng.randrange(B)] = -1
    return n


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bf16(gen, *shape, scale=1.0):
    out = torch.empty(*shape, dtype=torch.bfloat16, device="cuda")
    flat = out.view(-1)
    step = 1 << 26                                                    # the fp32 numbers of a 1 GB cache are not held at once
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda") * scale)
    return out


def _pages(case, seq, new, gen, seed):
    """Page pools of both kinds with the rows stored so far, and the table that says whose page is where (-1: none yet)."""
    ps, B = case["page"], case["batch"]
    need = [-(-(s + n) // ps) for s, n in zip(seq, new)]
    width = max(need) + 2
    count = sum(need) + 5
    order = random.Random(seed).sample(range(count), count)
    table = np.full((B, width), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    k = _bf16(gen, count, case["hkv"], ps, D)
    v = _bf16(gen, count, case["hkv"], ps, D)
    return k, v, torch.from_numpy(table).cuda()


def prepare(case, seed):
    gen = _gen(seed)
    st = dict(case=case)
    B, T = case["batch"], case["tokens"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")                                                    # noqa: E731
    if case["op"] == "verify":
        V, n = case["vocab"], _drafts(case)
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        logits = torch.randn(B, T + 1, V, generator=gen, device="cuda") * 2.0
        hot = torch.randint(0, V, (B, T + 1, 4), generator=gen, device="cuda")
        logits.scatter_add_(2, hot, torch.rand(B, T + 1, 4, generator=gen, device="cuda") * 14.0)       # a few likely tokens, as a model has them
        if case["dtype"] == "fp32" and V > 64:                        # processed scores: what a filter took out is -inf
            logits.masked_fill_(logits < -4.0, float("-inf"))
        logits = logits.to(dt)
        st["logits"] = logits
        st["n_draft"] = i32(n)
        st["u"] = torch.rand(B, T + 1, generator=gen, device="cuda")
        best = logits[:, :T].float().argmax(-1)
        other = torch.randint(0, V, (B, T), generator=gen, device="cuda")
        lucky = torch.rand(B, T, generator=gen, device="cuda") < 0.8
        st["drafts"] = torch.where(lucky, best, other)
        st["probs"] = None
        if case["probs"]:                                             # a draft model that is nearly right
            noisy = logits[:, :T].float() + torch.randn(B, T, V, generator=gen, device="cuda")
            st["probs"] = torch.softmax(noisy / max(case["temperature"], 0.3), -1)
            if T:
                drawn = torch.multinomial(st["probs"].view(B * T, V), 1, generator=gen).view(B, T)
                st["drafts"] = torch.where(lucky, drawn, other)
        st["accepted"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        st["tokens"] = torch.full((B, T + 1), -1, dtype=torch.int64, device="cuda")
        if own:
            st["ws"] = _ops().verify_drafts_workspace(B, T, V)
        return st
    seq, new = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    st["k_pages"], st["v_pages"], st["table"] = _pages(case, seq, new, gen, seed)
    st["seq_len"], st["n_new"] = i32(seq), i32(new)
    if case["op"] == "append":
        st["qkv"] = _bf16(gen, B, T, (hq + 2 * hkv) * D)
        pos = st["seq_len"].double()[:, None] + torch.arange(T, device="cuda", dtype=torch.float64) + 11000.0 + seed % 1000
        freq = 1.0e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = pos[:, :, None] * freq
        st["cos"], st["sin"] = torch.cos(ang).to(torch.bfloat16), torch.sin(ang).to(torch.bfloat16)
        st["q_out"] = torch.zeros(B, T, hq, D, dtype=torch.bfloat16, device="cuda")
        if own:
            _ops()
        return st
    P = case["prefix"]
    st["q"] = _bf16(gen, B, T, hq, D, scale=1.5)
    st["k_prefix"] = _bf16(gen, hkv, P + 7, D)
    st["v_prefix"] = _bf16(gen, hkv, P + 7, D)
    st["out"] = torch.zeros(B, T, hq, D, dtype=torch.bfloat16, device="cuda")
    if own:
        st["ws"] = _ops().batch_attn_workspace(B, T, P, st["table"].shape[1] * case["page"], hq, hkv)
    return st


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attn": _own_attn, "verify": _own_verify}[op](state)
    return {"append": _plain_append, "attn": _plain_attn, "verify": _plain_verify}[op](state)


def _own_append(s):
    c = s["case"]
    _ops().batch_rope_append(s["qkv"], s["cos"], s["sin"], s["seq_len"], s["n_new"], s["table"], s["k_pages"], s["v_pages"], c["hq"], c["hkv"], D, s["q_out"])
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attn(s):
    c = s["case"]
    _ops().batch_attn(s["q"], s["k_prefix"], s["v_prefix"], s["k_prefix"].stride(0), c["prefix"], s["k_pages"], s["v_pages"], s["table"], s["seq_len"],
                      s["n_new"], c["hq"], c["hkv"], D, D ** -0.5, s["out"], s["ws"])
    return {"out": s["out"]}


def _own_verify(s):
    _ops().verify_drafts(s["logits"], s["drafts"], s["n_draft"], s["probs"], s["u"], s["case"]["temperature"], s["accepted"], s["tokens"], s["ws"])
    return {"accepted": s["accepted"], "tokens": s["tokens"]}


def _plain_append(s):
    c = s["case"]
    B, T, hq, hkv, ps = c["batch"], c["tokens"], c["hq"], c["hkv"], c["page"]
    x = s["qkv"].view(B, T, hq + 2 * hkv, D)
    rot = x[:, :, :hq + hkv].float()
    cos, sin = s["cos"].float()[:, :, None], s["sin"].float()[:, :, None]
    lo, hi = rot[..., :D // 2], rot[..., D // 2:]
    y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(torch.bfloat16)
    t = torch.arange(T, device="cuda")
    live = t < s["n_new"][:, None]
    j = (s["seq_len"][:, None] + t).long()
    page = torch.gather(s["table"], 1, (j // ps).clamp(max=s["table"].shape[1] - 1)).long()
    b, tt = torch.nonzero(live, as_tuple=True)
    s["q_out"][b, tt] = y[b, tt, :hq]
    s["k_pages"][page[b, tt], :, j[b, tt] % ps] = y[b, tt, hq:]
    s["v_pages"][page[b, tt], :, j[b, tt] % ps] = x[b, tt, hq + hkv:]
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attn(s):
    c = s["case"]
    B, T, hq, hkv, P, ps = c["batch"], c["tokens"], c["hq"], c["hkv"], c["prefix"], c["page"]
    G, L = hq // hkv, s["table"].shape[1] * c["page"]
    t = torch.arange(T, device="cuda")
    live = t < s["n_new"][:, None]                                                         # [B, T]
    seen = torch.arange(L, device="cuda") <= (s["seq_len"][:, None] + t)[:, :, None]       # [B, T, L]
    table = s["table"].clamp(min=0).long()
    for h in range(hkv):
        q = s["q"][:, :, h * G:(h + 1) * G].float() * D ** -0.5                            # [B, T, G, D]
        far = torch.matmul(q.reshape(B * T * G, D), s["k_prefix"][h, :P].float().t())      # [rows, P]
        k = s["k_pages"][table, h].view(B, L, D).float()
        v = s["v_pages"][table, h].view(B, L, D).float()
        near = torch.matmul(q.view(B, T * G, D), k.transpose(1, 2)).view(B, T, G, L)
        near = near.masked_fill(~seen[:, :, None], float("-inf")).view(B * T * G, L)
        top = near.amax(-1, keepdim=True)
        if P:
            top = torch.maximum(top, far.amax(-1, keepdim=True))
        far, near = torch.exp(far - top), torch.exp(near - top)
        total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
        v = v.masked_fill(~seen.any(1)[:, :, None], 0.0)
        o = torch.matmul(far, s["v_prefix"][h, :P].float()) + torch.matmul(near.view(B, T * G, L), v).view(B * T * G, D)
        o = (o / total).view(B, T, G, D).to(torch.bfloat16)
        s["out"][:, :, h * G:(h + 1) * G] = torch.where(live[:, :, None, None], o, s["out"][:, :, h * G:(h + 1) * G])
    return {"out": s["out"]}


def _plain_verify(s):
    """In 64 bits: a token turns on whether a running sum of 150 000 terms passes a given number."""
    c = s["case"]
    B, T, V, temp = c["batch"], c["tokens"], c["vocab"], c["temperature"]
    x = s["logits"].double()
    n, drafts = s["n_draft"].long(), s["drafts"]
    t = torch.arange(T, device="cuda")
    if temp == 0:
        best = x.argmax(-1)                                                                # [B, T+1]
        ok = (drafts == best[:, :T]) & (t < n[:, None])
        taken = ok.long().cumprod(-1).sum(-1)
        last = best.gather(1, taken[:, None])[:, 0]
    else:
        x = (x - x.amax(-1, keepdim=True)) / temp
        e = torch.exp(x)
        p = e / e.sum(-1, keepdim=True)
        at = p[:, :T].gather(2, drafts[:, :, None])[:, :, 0]
        q = s["probs"].double() if s["probs"] is not None else None
        qx = q.gather(2, drafts[:, :, None])[:, :, 0] if q is not None else torch.ones_like(at)
        ok = (s["u"][:, :T].double() * qx < at) & (t < n[:, None])
        taken = ok.long().cumprod(-1).sum(-1)
        row = p.gather(1, taken[:, None, None].expand(B, 1, V))[:, 0]
        if T:
            refused = taken < n
            a = taken.clamp(max=T - 1)[:, None]
            if q is not None:
                less = q.gather(1, a[:, :, None].expand(B, 1, V))[:, 0]
            else:
                less = torch.zeros_like(row).scatter_(1, drafts.gather(1, a), 1.0)
            rest = (row - less).clamp(min=0.0)
            row = torch.where((refused & (rest.sum(-1) > 0))[:, None], rest, row)
        run_sum = row.cumsum(-1)
        over = (run_sum > s["u"][:, T:].double() * run_sum[:, -1:]) & (row > 0)
        last = torch.where(over.any(-1), over.long().argmax(-1), V - 1 - (row > 0).flip(-1).long().argmax(-1))
    busy = n >= 0
    col = torch.arange(T + 1, device="cuda")
    padded = torch.cat([drafts, drafts.new_zeros(B, 1)], 1)
    tokens = torch.where(col < taken[:, None], padded, torch.where(col == taken[:, None], last[:, None], torch.full_like(padded, -1)))
    s["tokens"].copy_(torch.where(busy[:, None], tokens, torch.full_like(tokens, -1)))
    s["accepted"].copy_(torch.where(busy, taken, torch.zeros_like(taken)))
    return {"accepted": s["accepted"], "tokens": s["tokens"]}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "verify": _exact_verify}[case["op"]](s)


def _exact_append(s):
    c = s["case"]
    hq, hkv, ps = c["hq"], c["hkv"], c["page"]
    q, k, v = s["q_out"].double(), s["k_pages"].double(), s["v_pages"].double()
    seq, new = _lengths(c)
    table = s["table"].cpu().numpy()
    half = D // 2
    for b in range(c["batch"]):
        for t in range(new[b]):
            heads = s["qkv"][b, t].double().view(hq + 2 * hkv, D)
            z = torch.complex(heads[:hq + hkv, :half], heads[:hq + hkv, half:]) * torch.complex(s["cos"][b, t].double(), s["sin"][b, t].double())
            turned = torch.cat([z.real, z.imag], -1)
            page, slot = int(table[b, (seq[b] + t) // ps]), (seq[b] + t) % ps
            q[b, t] = turned[:hq]
            k[page, :, slot] = turned[hq:]
            v[page, :, slot] = heads[hq + hkv:]
    return {"q": q, "k_pages": k, "v_pages": v}


def _exact_attn(s):
    c = s["case"]
    hq, hkv, P, ps = c["hq"], c["hkv"], c["prefix"], c["page"]
    G = hq // hkv
    out = s["out"].double()
    seq, new = _lengths(c)
    for h in range(hkv):
        kp, vp = s["k_prefix"][h, :P].double(), s["v_prefix"][h, :P].double()
        for b in range(c["batch"]):
            if new[b] == 0:
                continue
            n = seq[b] + new[b]
            pages = s["table"][b, :-(-n // ps)].long()
            ko = s["k_pages"][pages, h].reshape(-1, D)[:n].double()
            vo = s["v_pages"][pages, h].reshape(-1, D)[:n].double()
            qs = s["q"][b, :new[b], h * G:(h + 1) * G].double().transpose(0, 1)                     # [G, new, D]
            score = torch.cat([qs @ kp.t(), qs @ ko.t()], -1) / math.sqrt(D)
            score[:, :, P:] += torch.triu(torch.full((new[b], n), float("-inf"), dtype=torch.float64, device="cuda"), seq[b] + 1)
            w = torch.softmax(score, -1)
            out[b, :new[b], h * G:(h + 1) * G] = (w[:, :, :P] @ vp + w[:, :, P:] @ vo).transpose(0, 1)
    return {"out": out}


def _exact_verify(s):
    c = s["case"]
    T, V, temp = c["tokens"], c["vocab"], c["temperature"]
    accepted, tokens = [], []
    for b, n in enumerate(_drafts(c)):
        line, taken = [-1] * (T + 1), 0
        if n >= 0:
            drafts = s["drafts"][b].tolist()
            u = s["u"][b].double().tolist()
            while True:
                x = s["logits"][b, taken].double().cpu().numpy()
                if temp == 0:
                    last = int(np.argmax(x))
                    if taken < n and drafts[taken] == last:
                        line[taken], taken = last, taken + 1
                        continue
                    break
                p = np.exp((x - x.max()) / temp)
                p /= p.sum()
                if taken < n:
                    q = np.zeros(V)
                    if s["probs"] is None:
                        q[drafts[taken]] = 1.0
                    else:
                        q = s["probs"][b, taken].double().cpu().numpy()
                    if u[taken] * q[drafts[taken]] < p[drafts[taken]]:
                        line[taken], taken = drafts[taken], taken + 1
                        continue
                    rest = np.maximum(p - q, 0.0)
                    p = rest if rest.sum() > 0 else p
                upto = np.cumsum(p)
                able = np.flatnonzero(p > 0)
                hit = able[upto[able] > u[T] * upto[-1]]
                last = int(hit[0]) if len(hit) else int(able[-1])
                break
            line[taken] = last
        accepted.append(taken)
        tokens.append(line)
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(tokens, dtype=torch.int64)}


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once; the video's keys and values once for the whole batch."""
    if case["op"] == "verify":
        V, size = case["vocab"], 2 if case["dtype"] == "bf16" else 4
        n = [x for x in _drafts(case) if x >= 0]
        nbytes = sum((x + 1) * V * size + 16 * (x + 1) for x in n) + 8 * case["batch"] * (case["tokens"] + 2)
        if case["probs"] and case["temperature"]:
            nbytes += 4 * V * sum(x > 0 for x in n)                   # the draft's row at the refusal
        return {"bytes": nbytes, "flops": 3 * V * sum(x + 1 for x in n)}
    seq, new = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    rows = sum(new)
    if case["op"] == "append":
        return {"bytes": rows * 2 * D * (2 * (hq + 2 * hkv) + 1) + 8 * case["batch"], "flops": rows * (hq + hkv) * D * 3}
    keys = hkv * 4 * D * (case["prefix"] + sum(s + n for s, n in zip(seq, new) if n))
    pairs = sum(case["prefix"] + s + t + 1 for s, n in zip(seq, new) for t in range(n))
    return {"bytes": keys + rows * hq * D * 4 + 4 * sum(-(-(s + n) // case["page"]) for s, n in zip(seq, new)), "flops": 4 * D * hq * pairs}
