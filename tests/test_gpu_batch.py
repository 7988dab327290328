"""The operators that decode a batch over one prefilled video (qp_batch_rope_append, qp_batch_attn, qp_verify_drafts) against plain 64-bit
restatements of their definitions, at the sizes, masks and tables where they can go wrong.

Tolerances (half a step of bf16 is 2^-8 of a value, of fp32 2^-24):
  append   one rounding to bf16 of a sum whose two products are exact in fp32: 2^-8 |y| + 2^-23 (|x cos| + |x' sin|)
  attn     each probability is rounded to bf16 once (2^-8), the result once (2^-8); a weight exp2(c s - c m) carries the error of its exponent:
           the 128 products of a score summed in fp32 (128 * 2^-24 of sum |q k|), the products with c (2^-24 of c |s| and of c |m|, and of the
           fma) and 2^-21 of the exponential itself; the sum of n weights n 2^-24 at most, and the same again in the normaliser:
           2^-8 |o| + (2^-8 + 2 d + 4 n 2^-24) sum w |v|,   d = scale (2^-17 max sum |q k| + 2^-22 max |s|) + 2^-21
  verify   whole numbers: equal"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def ops():
    from quickvideo_amd.native import QuickPrefillOps
    return QuickPrefillOps(torch.device("cuda:0"))


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Pages, tables and lengths of a batch; every page row that nobody stored is NaN."""

    def __init__(self, hkv, ps, seq_len, n_new, t_max, seed, spare=3, width=None, gap=0):
        self.g = torch.Generator().manual_seed(seed)
        self.hkv, self.ps, self.B, self.T = hkv, ps, len(seq_len), t_max
        self.seq, self.new = list(seq_len), [max(0, min(n, t_max)) for n in n_new]
        need = [-(-(s + n) // ps) for s, n in zip(self.seq, self.new)]
        count = sum(need) + spare
        self.width = width or max(max(need), 1)
        order = torch.randperm(count, generator=self.g).tolist()
        self.table = np.full((self.B, self.width), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(need):
            n = min(n, self.width)
            self.table[b, :n] = order[at:at + n]
            at += n
        page = hkv * ps * D
        self.k_pool = torch.full((count, page + gap), float("nan"), dtype=torch.bfloat16)
        self.v_pool = torch.full((count, page + gap), float("nan"), dtype=torch.bfloat16)
        self.count, self.page = count, page

    def randn(self, *shape, scale=1.0):
        return (torch.randn(*shape, generator=self.g) * scale).to(torch.bfloat16)

    def view(self, pool):
        return pool[:, :self.page].unflatten(1, (self.hkv, self.ps, D))

    def row(self, pool, b, j):
        return self.view(pool)[int(self.table[b, j // self.ps]), :, j % self.ps]

    def fill(self, upto, scale=1.0):
        for b in range(self.B):
            for j in range(upto[b]):
                if j // self.ps < self.width and 0 <= self.table[b, j // self.ps] < self.count:
                    self.row(self.k_pool, b, j).copy_(self.randn(self.hkv, D, scale=scale))
                    self.row(self.v_pool, b, j).copy_(self.randn(self.hkv, D))

    def cuda(self):
        """(k_pages, v_pages, table, seq_len, n_new) on the device; the pages keep their distance."""
        k, v = self.k_pool.cuda(), self.v_pool.cuda()
        return self.view(k), self.view(v), torch.from_numpy(self.table).cuda(), i32(self.seq), i32(self.new)


# ------------------------------------------------------------------------------------------------------------------------------ append
def tables(g, B, T, base=11000):
    pos = base + torch.randint(0, 50000, (B, T), generator=g).double()
    ang = pos[:, :, None] * (1.0e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return torch.cos(ang).to(torch.bfloat16), torch.sin(ang).to(torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,ps,seq,new,T,gap", [
    (28, 4, 16, [11], [1], 1, 0), (28, 4, 16, [0], [1], 1, 0), (28, 4, 16, [15, 16, 17, 0], [1, 1, 1, 1], 1, 0), (64, 8, 24, [40, 0, 23, 5], [31, 0, 7, 48], 48, 0),
    (12, 2, 1, [3, 0], [2, 3], 3, 0), (7, 7, 5, [4, 9, 0], [3, 1, 2], 4, 0), (8, 1, 100, [99, 300], [2, 2], 2, 128), (1, 1, 7, [6], [9], 9, 8), (33, 11, 16, [2], [5], 6, 0),
    (28, 4, 64, [63] * 40, [1] * 40, 1, 0),
])
def test_append(ops, hq, hkv, ps, seq, new, T, gap):
    bt = Batch(hkv, ps, seq, new, T, seed=hq + ps, gap=gap)
    bt.fill(seq)
    B = bt.B
    cos, sin = tables(bt.g, B, T)
    qkv = bt.randn(B, T, (hq + 2 * hkv) * D)
    kp, vp, table, sl, nn = bt.cuda()
    k0, v0 = kp.clone(), vp.clone()
    q_out = torch.full((B, T, hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.batch_rope_append(qkv.cuda(), cos.cuda(), sin.cuda(), sl, nn, table, kp, vp, hq, hkv, D, q_out)
    x, c, s = f64(qkv).reshape(B, T, hq + 2 * hkv, D), f64(cos)[:, :, None], f64(sin)[:, :, None]
    lo, hi = x[..., :64], x[..., 64:]
    y = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    tol = 2.0 ** -8 * np.abs(y) + 2.0 ** -23 * np.concatenate([np.abs(lo * c) + np.abs(hi * s), np.abs(hi * c) + np.abs(lo * s)], -1)
    got_q, got_k, got_v = f64(q_out), f64(kp), f64(vp)
    want_k, want_v = f64(k0), f64(v0)
    tol_k = np.zeros_like(want_k)
    for b in range(B):
        for t in range(T):
            if t >= bt.new[b]:
                assert np.isnan(got_q[b, t]).all()                       # rows behind a sequence's last one are left alone
                continue
            assert (np.abs(got_q[b, t] - y[b, t, :hq]) <= tol[b, t, :hq]).all()
            page, slot = bt.table[b, (bt.seq[b] + t) // ps], (bt.seq[b] + t) % ps
            want_k[page, :, slot], tol_k[page, :, slot] = y[b, t, hq:hq + hkv], tol[b, t, hq:hq + hkv]
            want_v[page, :, slot] = x[b, t, hq + hkv:]
    assert np.array_equal(got_v, want_v, equal_nan=True)
    assert np.array_equal(np.isnan(got_k), np.isnan(want_k))
    assert (np.abs(got_k - want_k)[~np.isnan(want_k)] <= tol_k[~np.isnan(want_k)]).all()


def test_append_without_counts_and_with_counts_out_of_range(ops):
    """n_new None = t_max for all; numbers outside [0, t_max] are clamped."""
    bt = Batch(2, 8, [3, 5, 0], [4, 4, 4], 4, seed=5)
    bt.fill(bt.seq)
    cos, sin = tables(bt.g, 3, 4)
    qkv = bt.randn(3, 4, 8 * D).cuda()
    kp, vp, table, sl, _ = bt.cuda()
    outs = []
    for nn in (None, i32([4, 9, 2 ** 31 - 1])):
        k, v, q = kp.clone(), vp.clone(), torch.zeros(3, 4, 4, D, dtype=torch.bfloat16, device="cuda")
        ops.batch_rope_append(qkv, cos.cuda(), sin.cuda(), sl, nn, table, k, v, 4, 2, D, q)
        outs.append((k, v, q))
    for a, b in zip(*outs):
        assert np.array_equal(f64(a), f64(b), equal_nan=True)
    k, v, q = kp.clone(), vp.clone(), torch.zeros(3, 4, 4, D, dtype=torch.bfloat16, device="cuda")
    ops.batch_rope_append(qkv, cos.cuda(), sin.cuda(), sl, i32([-5, 0, -2 ** 31]), table, k, v, 4, 2, D, q)
    assert np.array_equal(f64(k), f64(kp), equal_nan=True) and np.array_equal(f64(v), f64(vp), equal_nan=True) and not q.any()


@pytest.mark.parametrize("bad", [-1, 7, 2 ** 31 - 1, -2 ** 31])
def test_append_follows_no_bad_page(ops, bad):
    """A page number out of range, a row behind the table and a negative length are dropped; the queries come out all the same."""
    bt = Batch(2, 4, [2, 6, 0, 0], [3, 3, 3, 3], 3, seed=6, spare=0, width=2)
    assert bt.count == 7
    bt.table[0, 1] = bad                                    # rows 4 of sequence 0
    bt.seq[2] = -2                                          # rows -2, -1 nowhere, row 0 stored
    kp, vp, table, sl, nn = bt.cuda()
    cos, sin = tables(bt.g, 4, 3)
    qkv = bt.randn(4, 3, 8 * D)
    q = torch.full((4, 3, 4, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.batch_rope_append(qkv.cuda(), cos.cuda(), sin.cuda(), sl, nn, table, kp, vp, 4, 2, D, q)
    assert torch.isfinite(q.float()).all()
    v = f64(vp)
    want = np.full_like(v, np.nan)
    x = f64(qkv).reshape(4, 3, 8, D)
    for b, t, j in [(0, 0, 2), (0, 1, 3), (1, 0, 6), (1, 1, 7), (2, 2, 0), (3, 0, 0), (3, 1, 1), (3, 2, 2)]:
        want[bt.table[b, j // 4], :, j % 4] = x[b, t, 6:]
    assert np.array_equal(v, want, equal_nan=True)


def test_append_agrees_with_the_prefill_append(ops):
    """Where qp_rope_append rounds after each step, the keys differ from its keys by no more than those steps do (3 half steps of the products
    and the sum), and the values not at all."""
    hq, hkv, n = 28, 4, 50
    bt = Batch(hkv, 16, [0], [n], n, seed=9)
    kp, vp, table, sl, nn = bt.cuda()
    qkv = bt.randn(1, n, (hq + 2 * hkv) * D).cuda()
    pos = torch.arange(n).repeat(3, 1).contiguous().cuda() + 4000
    cos, sin = ops.mrope_table(pos, (16, 24, 24), 1e6, D)
    q, q2 = torch.empty(1, n, hq, D, dtype=torch.bfloat16, device="cuda"), torch.empty(n, hq, D, dtype=torch.bfloat16, device="cuda")
    k2, v2 = (torch.empty(hkv, n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.batch_rope_append(qkv, cos, sin, sl, nn, table, kp, vp, hq, hkv, D, q)
    ops.rope_append(qkv[0], cos, sin, hq, hkv, D, q2, k2, v2, n * D, 0, None)
    idx = table[0].long()
    k1 = kp[idx].transpose(1, 2).reshape(-1, hkv, D)[:n].transpose(0, 1)
    v1 = vp[idx].transpose(1, 2).reshape(-1, hkv, D)[:n].transpose(0, 1)
    assert torch.equal(v1, v2)
    size = 2 * qkv.float().abs().max().item()
    assert (k1.float() - k2.float()).abs().max().item() <= 4 * 2.0 ** -8 * size
    assert (q[0].float() - q2.float()).abs().max().item() <= 4 * 2.0 ** -8 * size


# --------------------------------------------------------------------------------------------------------------------------- attention
def attn_ref(q, kpre, vpre, P, bt, hq, scale):
    """64 bits: (out, tolerance) [B, T, hq, D], NaN where nothing is written."""
    B, T, hkv = bt.B, bt.T, bt.hkv
    G = hq // hkv
    out, tol = np.full((B, T, hq, D), np.nan), np.zeros((B, T, hq, D))
    q = f64(q)
    for h in range(hkv):
        kp, vp = (f64(kpre[h, :P]), f64(vpre[h, :P])) if P else (np.zeros((0, D)),) * 2
        for b in range(B):
            rows = [j for j in range(min(bt.seq[b] + bt.new[b], bt.width * bt.ps)) if 0 <= bt.table[b, j // bt.ps] < bt.count]
            kb = np.stack([f64(bt.row(bt.k_pool, b, j)[h]) for j in rows]) if rows else np.zeros((0, D))
            vb = np.stack([f64(bt.row(bt.v_pool, b, j)[h]) for j in rows]) if rows else np.zeros((0, D))
            for t in range(bt.new[b]):
                see = [i for i, j in enumerate(rows) if j <= bt.seq[b] + t]
                k, v = np.concatenate([kp, kb[see]]), np.concatenate([vp, vb[see]])
                o_rows = q[b, t, h * G:(h + 1) * G]
                if len(k) == 0:
                    out[b, t, h * G:(h + 1) * G] = 0.0
                    continue
                with np.errstate(all="ignore"):
                    s = o_rows @ k.T * scale
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    o = w @ v
                    d = 2.0 ** -17 * scale * (np.abs(o_rows) @ np.abs(k).T).max(-1, keepdims=True) + 2.0 ** -22 * np.abs(s).max(-1, keepdims=True) + 2.0 ** -21
                    out[b, t, h * G:(h + 1) * G] = o
                    tol[b, t, h * G:(h + 1) * G] = 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + 2 * d + 4 * len(k) * 2.0 ** -24) * (w @ np.abs(v))
    return out, tol


def run_attn(ops, q, kpre, vpre, P, bt, hq, scale, n_new="given", out=None):
    kp, vp, table, sl, nn = bt.cuda()
    B, T = bt.B, bt.T
    ws = ops.batch_attn_workspace(B, T, P, bt.width * bt.ps, hq, bt.hkv)
    ws.fill_(255)                                                        # NaN patterns: a partial result that was not written must not count
    if out is None:
        out = torch.full((B, T, hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.batch_attn(q, kpre, vpre, kpre.stride(0) if kpre is not None else 0, P, kp, vp, table, sl, nn if n_new == "given" else n_new, hq, bt.hkv, D, scale, out, ws)
    return out


def check(got, ref, tol):
    got = f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), "NaN in other places"
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf])
    ok = ~np.isnan(ref) & ~inf
    bad = np.abs(got[ok] - ref[ok]) - tol[ok]
    assert (bad <= 0).all(), bad.max()


def prefix_of(bt, P, scale=1.0, room=5):
    k, v = torch.full((bt.hkv, P + room, D), float("nan"), dtype=torch.bfloat16), torch.full((bt.hkv, P + room, D), float("nan"), dtype=torch.bfloat16)
    k[:, :P], v[:, :P] = bt.randn(bt.hkv, P, D, scale=scale), bt.randn(bt.hkv, P, D)
    return k.cuda(), v.cuda()


ATTN = [  # hq, hkv, P, page, seq_len, n_new, t_max
    (28, 4, 0, 16, [0], [1], 1), (28, 4, 1, 16, [0], [1], 1), (28, 4, 63, 16, [5], [1], 1), (28, 4, 64, 16, [64], [1], 1), (28, 4, 65, 16, [63, 127], [1, 1], 1),
    (12, 2, 417, 16, [9], [1], 1), (64, 8, 1000, 32, [250, 0, 31], [6, 0, 2], 6), (8, 1, 4097, 7, [100, 3, 0], [3, 3, 1], 3), (7, 7, 130, 1, [17, 40], [5, 2], 5),
    (32, 2, 777, 24, [0, 70], [4, 4], 4), (40, 1, 300, 100, [99], [2], 2), (28, 4, 515, 16, [5, 0, 9, 2], [61, 1, 0, 30], 61), (16, 16, 33, 128, [200], [1], 1),
    (28, 4, 2049, 16, [3, 900, 40, 0, 77, 512, 1, 64], [1] * 8, 1), (28, 4, 0, 5, [300, 12], [17, 40], 40), (14, 2, 129, 16, list(range(0, 90, 3)), [1] * 30, 1),
    (28, 4, 0, 16, [1500], [1], 1), (4, 1, 6001, 16, [2], [129], 129),
]


@pytest.mark.parametrize("hq,hkv,P,ps,seq,new,T", ATTN)
def test_attn(ops, hq, hkv, P, ps, seq, new, T):
    bt = Batch(hkv, ps, seq, new, T, seed=P + hq)
    bt.fill([s + n for s, n in zip(bt.seq, bt.new)])
    kpre, vpre = prefix_of(bt, P)
    q = bt.randn(bt.B, T, hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    qd = q.cuda()
    got = run_attn(ops, qd, kpre, vpre, P, bt, hq, D ** -0.5)
    check(got, ref, tol)
    again = run_attn(ops, qd, kpre, vpre, P, bt, hq, D ** -0.5)          # no order that changes: the same bits
    assert np.array_equal(f64(got), f64(again), equal_nan=True)


@pytest.mark.parametrize("hq,hkv,P,ps,seq,T", [
    (8, 1, 500, 16, [3, 0], 62), (7, 7, 1030, 16, [30, 5, 0], 40), (28, 4, 1024, 24, [9, 100], 128), (4, 2, 2000, 16, [0], 129), (12, 2, 700, 16, list(range(100)), 1),
    (16, 1, 4100, 16, [7], 300), (6, 3, 999, 1, [2, 1, 4], 32),
])
def test_attn_full_batches_of_many_tokens(ops, hq, hkv, P, ps, seq, T):
    """n_new None: many tokens over a longer prefix go through the prefill kernel, head by head (its probabilities are rounded once: within the bound)."""
    bt = Batch(hkv, ps, seq, [T] * len(seq), T, seed=P)
    bt.fill([s + T for s in seq])
    kpre, vpre = prefix_of(bt, P)
    q = bt.randn(bt.B, T, hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=None), ref, tol)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5), ref, tol)


@pytest.mark.parametrize("hq,hkv,P,B,T", [(8, 2, 300, 100, 3), (4, 1, 700, 65, 9), (4, 2, 129, 600, 2), (2, 2, 64, 513, 3), (28, 4, 400, 5, 61), (4, 1, 2500, 512, 2)])
@pytest.mark.parametrize("fill", ["some", "one", "none"])
def test_attn_padded_batches(ops, hq, hkv, P, B, T, fill):
    """Most places of the batch empty: only the live tokens count, wherever they are."""
    rs = np.random.RandomState(B + T)
    new = rs.randint(0, T + 1, B) * (rs.rand(B) < 0.5) if fill == "some" else np.zeros(B, dtype=int)
    if fill == "one":
        new[B // 2] = T
    seq = rs.randint(0, 20, B)
    bt = Batch(hkv, 4, seq.tolist(), new.tolist(), T, seed=B)
    bt.fill([s + n for s, n in zip(bt.seq, bt.new)])
    kpre, vpre = prefix_of(bt, P)
    q = torch.full((B, T, hq, D), float("nan"), dtype=torch.bfloat16)               # what a dead row holds must not matter
    for b in range(B):
        q[b, :bt.new[b]] = bt.randn(bt.new[b], hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5), ref, tol)


@pytest.mark.parametrize("P", [50, 3000])
@pytest.mark.parametrize("T,B", [(1, 2), (5, 3), (70, 2)])
def test_attn_infinite_values_in_the_prefix(ops, P, T, B):
    """A value row of the prefix that is not finite reaches every row that sees it (all of them), through every form of the operator, and no other column."""
    for n_new in ("given", None):
        bt = Batch(2, 16, [5] * B, [T] * B, T, seed=T)
        bt.fill([5 + T] * B)
        kpre, vpre = prefix_of(bt, P)
        vpre[0, P // 2, 3] = float("inf"); vpre[1, P - 1, 100] = float("-inf"); vpre[1, 0, 7] = float("nan")
        q = bt.randn(B, T, 8, D)
        ref, tol = attn_ref(q, kpre, vpre, P, bt, 8, D ** -0.5)
        assert np.isinf(ref[:, :, :4, 3]).all() and np.isinf(ref[:, :, 4:, 100]).all() and np.isnan(ref[:, :, 4:, 7]).all() and np.isfinite(ref[:, :, :4, :3]).all()
        check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, 8, D ** -0.5, n_new=n_new), ref, tol)


@pytest.mark.parametrize("sigma,scale", [(0.0, D ** -0.5), (12.0, D ** -0.5), (150.0, D ** -0.5), (1.0, 3.0), (1.0, 1e-4)])
def test_attn_flat_and_peaked(ops, sigma, scale):
    """All scores equal; one key that takes everything; scores of thousands; other scales."""
    bt = Batch(2, 16, [40, 3], [5, 5], 5, seed=int(sigma) + 1)
    bt.fill([45, 8], scale=sigma)
    kpre, vpre = prefix_of(bt, 900, scale=sigma)
    q = bt.randn(2, 5, 14, D)
    ref, tol = attn_ref(q, kpre, vpre, 900, bt, 14, scale)
    check(run_attn(ops, q.cuda(), kpre, vpre, 900, bt, 14, scale), ref, tol)


@pytest.mark.parametrize("T,where", [(1, 0), (4, 0), (4, 2), (30, 1)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_attn_masked_rows_may_hold_anything(ops, T, where, value):
    """Key and value rows of drafted token `where` hold non-finite numbers: the tokens before it must not notice, the ones behind it get what the
    definition gives them (values: infinity or NaN through the sum; keys: a NaN or infinite score)."""
    for what in ("v", "k"):
        bt = Batch(2, 16, [37, 62], [T, T], T, seed=T)
        bt.fill([37 + T, 62 + T])
        row = bt.row(bt.v_pool if what == "v" else bt.k_pool, 1, 62 + where)
        row[:, 5] = value
        row[1, 77] = -value
        kpre, vpre = prefix_of(bt, 200)
        q = bt.randn(2, T, 8, D).abs()
        ref, tol = attn_ref(q, kpre, vpre, 200, bt, 8, D ** -0.5)
        assert np.isfinite(ref[1, :where]).all() and np.isfinite(ref[0]).all() and not np.isfinite(ref[1, where:]).all()
        check(run_attn(ops, q.cuda(), kpre, vpre, 200, bt, 8, D ** -0.5), ref, tol)


@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1, -2 ** 31, 12])
def test_attn_follows_no_bad_page_and_a_row_without_keys_is_zero(ops, bad):
    bt = Batch(2, 4, [13, 3, 0], [3, 3, 2], 3, seed=4, spare=0)
    bt.fill([16, 6, 2])
    pages = bt.table.copy()
    bt.table[0, 1] = bad if bad != 12 else bt.count         # a hole in the middle
    bt.table[1, 0] = bad if bad != 12 else bt.count         # rows 0..3 gone: token 0 sees nothing of its own
    bt.table[2, 0] = bad if bad != 12 else bt.count         # nothing at all
    q = bt.randn(3, 3, 6, D)
    for P in (0, 70):
        kpre, vpre = prefix_of(bt, P)
        ref, tol = attn_ref(q, kpre, vpre, P, bt, 6, D ** -0.5)
        if P == 0:
            assert not ref[2, :2].any() and not ref[1, 0].any()
        check(run_attn(ops, q.cuda(), kpre if P else None, vpre if P else None, P, bt, 6, D ** -0.5), ref, tol)
    bt.table[:] = pages


def test_attn_lengths_out_of_range(ops):
    """Lengths behind the table are cut to it, negative ones leave what is visible; n_new is clamped; None = all."""
    bt = Batch(2, 8, [20, 20, 5], [3, 3, 3], 3, seed=8, width=3)
    bt.fill([23, 23, 8])
    kpre, vpre = prefix_of(bt, 100)
    q = bt.randn(3, 3, 8, D)
    bt.seq = [2 ** 31 - 1, 30, -2]                          # sequences 0, 1: all 24 rows of the table (23 stored + NaN row 23 refilled below)
    for b in (0, 1):
        bt.row(bt.k_pool, b, 23).copy_(bt.randn(2, D)); bt.row(bt.v_pool, b, 23).copy_(bt.randn(2, D))
    ref, tol = attn_ref(q, kpre, vpre, 100, bt, 8, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, 100, bt, 8, D ** -0.5), ref, tol)
    a = run_attn(ops, q.cuda(), kpre, vpre, 100, bt, 8, D ** -0.5, n_new=None)
    b = run_attn(ops, q.cuda(), kpre, vpre, 100, bt, 8, D ** -0.5, n_new=i32([3, 99, 2 ** 31 - 1]))
    assert torch.equal(a, b) and np.array_equal(f64(a), f64(run_attn(ops, q.cuda(), kpre, vpre, 100, bt, 8, D ** -0.5)))
    keep = torch.full_like(a, 7.0)
    c = run_attn(ops, q.cuda(), kpre, vpre, 100, bt, 8, D ** -0.5, n_new=i32([0, -4, -2 ** 31]), out=keep)
    assert (c == 7.0).all()


def test_attn_in_place(ops):
    bt = Batch(4, 16, [30, 4], [3, 2], 3, seed=12)
    bt.fill([33, 6])
    kpre, vpre = prefix_of(bt, 333)
    q = bt.randn(2, 3, 28, D)
    want = run_attn(ops, q.cuda(), kpre, vpre, 333, bt, 28, D ** -0.5)
    qd = q.cuda()
    got = run_attn(ops, qd, kpre, vpre, 333, bt, 28, D ** -0.5, out=qd)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :2], want[1, :2]) and torch.equal(got[1, 2].cpu(), q[1, 2])


def test_attn_shared_pages_and_interleaved_pools(ops):
    """Two sequences read the same page (a forked answer), K and V pages lie between one another in one buffer."""
    bt = Batch(2, 8, [16, 16, 9], [1, 1, 1], 1, seed=13)
    bt.fill([17, 17, 10])
    bt.table[1, :2] = bt.table[0, :2]
    kpre, vpre = prefix_of(bt, 50)
    q = bt.randn(3, 1, 4, D)
    ref, tol = attn_ref(q, kpre, vpre, 50, bt, 4, D ** -0.5)
    both = torch.stack([bt.view(bt.k_pool), bt.view(bt.v_pool)], 1).cuda()          # [pages, 2, hkv, ps, D]
    ws = ops.batch_attn_workspace(3, 1, 50, bt.width * 8, 4, 2)
    out = torch.empty(3, 1, 4, D, dtype=torch.bfloat16, device="cuda")
    ops.batch_attn(q.cuda(), kpre, vpre, kpre.stride(0), 50, both[:, 0], both[:, 1], torch.from_numpy(bt.table).cuda(), i32(bt.seq), None, 4, 2, D, D ** -0.5, out, ws)
    check(out, ref, tol)


def test_offsets_past_32_bits(ops):
    """Pages and prefix heads that lie more than 2^32 bytes (and 2^31 elements) from the start of their buffers."""
    hq, hkv, ps, far = 8, 2, 16, 600_000                     # page stride 2 * 16 * 128 * 2 B = 8 KB: page 600 000 at 4.9 GB
    P, cap = 90, 18_000_000                                  # head 1 starts at 2.3e9 elements = 4.6 GB
    g = torch.Generator().manual_seed(1)
    pool = torch.empty(far + 4, hkv, ps, D, dtype=torch.bfloat16, device="cuda")
    bt = Batch(hkv, ps, [20, 1], [2, 2], 2, seed=21, spare=0)
    small = bt.table.copy()
    remap = {int(p): far + i for i, p in enumerate(sorted(set(small[small >= 0].tolist())))}
    big = np.vectorize(lambda p: remap.get(int(p), -1))(small).astype(np.int32)
    bt.fill([20, 1])
    for p, where in remap.items():
        pool[where] = bt.view(bt.k_pool)[p].cuda()
    cos, sin = tables(g, 2, 2)
    qkv = bt.randn(2, 2, (hq + 2 * hkv) * D).cuda()
    kp, vp, table, sl, nn = bt.cuda()
    q1, q2 = (torch.empty(2, 2, hq, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.batch_rope_append(qkv, cos.cuda(), sin.cuda(), sl, nn, table, kp, vp, hq, hkv, D, q1)
    vpool = torch.empty_like(pool)
    for p, where in remap.items():
        vpool[where] = bt.view(bt.v_pool)[p].cuda()
    tb = torch.from_numpy(big).cuda()
    ops.batch_rope_append(qkv, cos.cuda(), sin.cuda(), sl, nn, tb, pool, vpool, hq, hkv, D, q2)
    assert torch.equal(q1, q2)
    for p, where in remap.items():
        assert np.array_equal(f64(pool[where]), f64(kp[p]), equal_nan=True) and np.array_equal(f64(vpool[where]), f64(vp[p]), equal_nan=True)
    kpre, vpre = prefix_of(bt, P)
    far_k = torch.empty(hkv, cap, D, dtype=torch.bfloat16, device="cuda")
    far_v = torch.empty(hkv, cap, D, dtype=torch.bfloat16, device="cuda")
    far_k[:, :P], far_v[:, :P] = kpre[:, :P], vpre[:, :P]
    ws = ops.batch_attn_workspace(2, 2, P, bt.width * ps, hq, hkv)
    o1, o2 = torch.empty_like(q1), torch.empty_like(q1)
    ops.batch_attn(q1, kpre, vpre, kpre.stride(0), P, kp, vp, table, sl, nn, hq, hkv, D, D ** -0.5, o1, ws)
    ops.batch_attn(q1, far_k, far_v, far_k.stride(0), P, pool, vpool, tb, sl, nn, hq, hkv, D, D ** -0.5, o2, ws)
    assert torch.equal(o1, o2)


def test_long_prefix_against_the_single_token_kernel(ops):
    """200 000 shared keys: every sequence gets what qp_decode_attn gives it over (prefix + its own rows) in one cache, within the two kernels' roundings
    (each: probabilities and result to bf16)."""
    hq, hkv, P, own = 28, 4, 200_003, 21
    g = torch.Generator(device="cuda").manual_seed(2)
    kpre = torch.randn(hkv, P + own, D, generator=g, device="cuda").to(torch.bfloat16)
    vpre = torch.randn(hkv, P + own, D, generator=g, device="cuda").to(torch.bfloat16)
    bt = Batch(hkv, 16, [own - 1] * 3, [1] * 3, 1, seed=3)
    bt.fill([own] * 3)
    q = bt.randn(3, 1, hq, D, scale=1.5)
    got = run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5)
    dws = ops.decode_attn_workspace(hq, hkv)
    for b in range(3):
        for j in range(own):
            kpre[:, P + j], vpre[:, P + j] = bt.row(bt.k_pool, b, j).cuda(), bt.row(bt.v_pool, b, j).cuda()
        one = torch.empty(hq, D, dtype=torch.bfloat16, device="cuda")
        ops.decode_attn(q[b, 0].cuda(), kpre, vpre, (P + own) * D, torch.tensor([P + own - 1, 0], device="cuda"), hq, hkv, D, D ** -0.5, one, dws)
        s = torch.einsum("hgd,hkd->hgk", q[b, 0].cuda().view(hkv, 7, D).float(), kpre.float()) * D ** -0.5
        size = torch.einsum("hgk,hkd->hgd", torch.softmax(s, -1), vpre.float().abs()).reshape(hq, D)
        assert ((got[b, 0].float() - one.float()).abs() <= 2 * 2.0 ** -8 * (one.float().abs() + size)).all()


# ------------------------------------------------------------------------------------------------------------------------- verification
def verify_ref(logits, drafts, n_draft, probs, u, temp):
    x = f64(logits)
    B, rows, V = x.shape
    T = rows - 1
    acc, tok = np.zeros(B, dtype=np.int64), np.full((B, rows), -1, dtype=np.int64)
    for b in range(B):
        n = T if n_draft is None else min(int(n_draft[b]), T)
        if n < 0:
            continue
        for a in range(n + 1):
            row = np.where(np.isnan(x[b, a]), -np.inf, x[b, a])
            m = row.max()
            none = m == -np.inf
            d = int(drafts[b, a]) if a < n else -1
            inside = 0 <= d < V
            if temp == 0:
                nxt = -1 if none else int(np.argmax(row))
                stands = inside and not none and d == nxt
            else:
                with np.errstate(all="ignore"):
                    w = np.where(row == m, 1.0, np.exp((row - m) / temp)) if not none else np.zeros(V)
                z = w.sum()
                q = None
                if a < n:
                    q = f64(probs[b, a]) if probs is not None else np.zeros(V)
                    if probs is None and inside:
                        q[d] = 1.0
                stands = inside and not none and float(u[b, a]) * q[d] * z < w[d]
            if a < n and stands:
                tok[b, a] = d
                continue
            acc[b] = a
            if temp != 0:
                r = w
                if a < n:
                    rest = np.where(np.isnan(q), 0.0, np.maximum(w - np.nan_to_num(q) * z, 0.0))
                    r = rest if rest.sum() > 0 else w
                can = np.flatnonzero(r > 0)
                upto = np.cumsum(r)
                hit = can[upto[can] > float(u[b, T]) * upto[-1]] if len(can) else can
                nxt = -1 if none else int(hit[0] if len(hit) else can[-1])
            tok[b, a] = nxt
            break
    return acc, tok


def run_verify(ops, logits, drafts, n_draft, probs, u, temp):
    B, rows, V = logits.shape
    ws = ops.verify_drafts_workspace(B, rows - 1, V)
    ws.fill_(255)
    acc = torch.full((B,), 77, dtype=torch.int32, device="cuda")
    tok = torch.full((B, rows), 77, dtype=torch.int64, device="cuda")
    ops.verify_drafts(logits, drafts.cuda(), None if n_draft is None else i32(n_draft), probs, None if u is None else u.cuda(), temp, acc, tok, ws)
    return acc.cpu().numpy(), tok.cpu().numpy()


def verify_case(B, T, V, dtype, with_probs, seed, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T + 1, V, generator=g) * sharp
    x[:, :, V // 3] += 9.0 * torch.rand(B, T + 1, generator=g)
    x = x.to(dtype)
    drafts = torch.where(torch.rand(B, T, generator=g) < 0.7, x[:, :T].float().argmax(-1), torch.randint(0, V, (B, T), generator=g))
    probs = torch.softmax(x[:, :T].float() + torch.randn(B, T, V, generator=g), -1) if with_probs else None
    u = torch.rand(B, T + 1, generator=g)
    return x, drafts, probs, u


@pytest.mark.parametrize("B,T,V", [(1, 0, 1), (1, 1, 1), (3, 2, 2), (2, 3, 3), (4, 4, 97), (2, 2, 4095), (2, 2, 4096), (2, 2, 4097), (1, 3, 151936), (5, 4, 152064), (40, 0, 1000),
                                   (2, 40, 300), (1, 255, 50)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0])
def test_verify(ops, B, T, V, dtype, with_probs, temp):
    x, drafts, probs, u = verify_case(B, T, V, dtype, with_probs, seed=V + T)
    n = [(-1 if B > 2 and b == 1 else (T - b) % (T + 1)) for b in range(B)]
    for n_draft in (None, n):
        want = verify_ref(x, drafts, n_draft, probs, u, temp)
        got = run_verify(ops, x.cuda(), drafts, n_draft, probs.cuda() if probs is not None else None, u, temp)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("temp", [1e-6, 0.05, 100.0])
@pytest.mark.parametrize("sharp", [0.0, 30.0])
def test_verify_temperatures(ops, temp, sharp):
    x, drafts, probs, u = verify_case(6, 3, 5000, torch.float32, True, seed=3, sharp=sharp)
    want = verify_ref(x, drafts, None, probs, u, temp)
    got = run_verify(ops, x.cuda(), drafts, None, probs.cuda(), u, temp)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_the_ends_of_the_random_numbers(ops, with_probs):
    """0 takes the first token that can be drawn, the largest number below 1 the last; 1 and more the last as well, below 0 the first, NaN refuses."""
    x, drafts, probs, u = verify_case(8, 3, 4500, torch.float32, with_probs, seed=5)
    x[:, :, :7] = float("-inf"); x[:, :, -9:] = float("-inf")
    if probs is not None:
        probs = torch.softmax(x[:, :3] * 0.9, -1)
    for val in (0.0, 1.0 - 2.0 ** -24, 1.0, 1.5, -0.5, float("nan")):
        for cols in ([3], [0], [0, 1, 2, 3]):
            u2 = u.clone()
            u2[:, cols] = val
            want = verify_ref(x, drafts, None, probs, u2, 0.8)
            got = run_verify(ops, x.cuda(), drafts, None, None if probs is None else probs.cuda(), u2, 0.8)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (val, cols)


def test_verify_odd_logits(ops):
    """-infinity, NaN and infinite logits; rows that offer nothing; drafts outside the vocabulary; equal distributions; a certain draft refused."""
    x, drafts, probs, u = verify_case(10, 2, 4200, torch.float32, True, seed=6)
    x[0] = float("-inf")
    x[1, 1] = float("nan")
    x[2, :, 100] = float("inf"); x[2, :, 4150] = float("inf")
    x[3, 0, 5] = float("nan"); drafts[3, 0] = 5
    drafts[4, 0] = -1; drafts[5, 0] = 4200; drafts[6, 1] = 2 ** 62
    probs[7] = torch.softmax(x[7, :2].double(), -1).float()
    probs[8, 0] = float("nan")
    u[9, 0] = 0.999999; x[9, 0] = -30.0; x[9, 0, 4199] = 12.0; drafts[9, 0] = 4199
    for p in (probs, None):
        for temp in (0.0, 0.6):
            want = verify_ref(x, drafts, None, p, u, temp)
            got = run_verify(ops, x.cuda(), drafts, None, None if p is None else p.cuda(), u, temp)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (p is None, temp)


def test_verify_greedy_ties_take_the_lowest_index(ops):
    x = torch.full((3, 2, 152064), 1.0, dtype=torch.bfloat16)
    x[1, 0, 5000] = x[1, 0, 100_000] = 2.0
    x[2, 0, 8191] = x[2, 0, 8192] = 2.0
    drafts = torch.tensor([[0], [5000], [8192]])
    got = run_verify(ops, x.cuda(), drafts, None, None, None, 0.0)
    assert got[0].tolist() == [1, 1, 0] and got[1].tolist() == [[0, 0], [5000, 0], [8191, -1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift,pad", [(0, 3), (1, 0), (3, 5), (7, 64)])
def test_verify_strided_and_unaligned(ops, dtype, shift, pad):
    """A slice of padded logits that starts at any element."""
    B, T, V = 3, 2, 9001
    x, drafts, probs, u = verify_case(B, T, V, dtype, True, seed=8)
    buf = torch.full((B * (T + 1) * (V + pad) + 16,), float("nan"), dtype=dtype, device="cuda")
    view = buf[shift:shift + B * (T + 1) * (V + pad)].view(B, T + 1, V + pad)[:, :, :V]
    view.copy_(x.cuda())
    pbuf = torch.full((B * T * (V + pad) + 16,), float("nan"), device="cuda")
    pview = pbuf[shift:shift + B * T * (V + pad)].view(B, T, V + pad)[:, :, :V]
    pview.copy_(probs.cuda())
    for temp in (0.0, 0.9):
        for p, pv in ((None, None), (probs, pview)):
            want = verify_ref(x, drafts, None, p, u, temp)
            got = run_verify(ops, view, drafts, None, pv, u, temp)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_draws_the_model_distribution(ops):
    """The point of the rule: over a fine grid of random numbers the first token comes out as the MODEL would have drawn it, whatever the draft's own
    distribution is.  300 x 300 grid: a count may be off by the cells a border crosses (at most one row and one column of the grid per token)."""
    N, V = 300, 5
    x = torch.tensor([1.0, 0.2, -0.7, 0.9, -3.0])
    q = torch.tensor([0.1, 0.5, 0.2, 0.15, 0.05])
    p = torch.softmax(x.double(), -1)
    grid = (torch.arange(N) + 0.5) / N
    u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).reshape(-1, 2).contiguous()
    total = torch.zeros(V, dtype=torch.float64)
    for d in range(V):                                                  # the draft model draws d with probability q[d]
        for lo in range(0, N * N, 60000):
            uu = u[lo:lo + 60000]
            B = len(uu)
            logits = x.expand(B, 2, V).contiguous().cuda()
            _, tok = run_verify(ops, logits, torch.full((B, 1), d), None, q.expand(B, 1, V).contiguous().cuda(), uu, 1.0)
            total += q[d].double() * torch.bincount(torch.from_numpy(tok[:, 0]), minlength=V).double() / (N * N)
    assert (total - p).abs().max().item() <= 2.0 * V / N


# --------------------------------------------------------------------------------------------------------- streams, graphs, all together
def test_on_another_stream(ops):
    bt = Batch(4, 16, [30, 4], [2, 2], 2, seed=31)
    bt.fill([32, 6])
    kpre, vpre = prefix_of(bt, 500)
    q = bt.randn(2, 2, 28, D).cuda()
    want = run_attn(ops, q, kpre, vpre, 500, bt, 28, D ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_attn(ops, q, kpre, vpre, 500, bt, 28, D ** -0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_step_replays_with_new_lengths(ops):
    """append -> attention -> verification captured once; before each replay lengths, counts, tables and inputs change.  Two graphs with workspaces of
    their own replay in turn, eager work and synchronisations between; every replay equals the eager call."""
    hq, hkv, ps, T, V, P = 28, 4, 16, 3, 5000, 300
    bt = Batch(hkv, ps, [60, 60], [T, T], T, seed=41)
    bt.fill([60, 60])
    kpre, vpre = prefix_of(bt, P)
    kp, vp, table, sl, nn = bt.cuda()
    g = torch.Generator().manual_seed(4)
    cos, sin = (t.cuda() for t in tables(g, 2, T))
    u = torch.rand(2, T, generator=g).cuda()

    class Step:
        def __init__(self):
            self.qkv = torch.zeros(2, T, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device="cuda")
            self.k, self.v, self.seq, self.new, self.table = kp.clone(), vp.clone(), sl.clone(), nn.clone(), table.clone()
            self.q = torch.zeros(2, T, hq, D, dtype=torch.bfloat16, device="cuda")
            self.out = torch.zeros_like(self.q)
            self.logits = torch.zeros(2, T, V, dtype=torch.float32, device="cuda")
            self.drafts, self.nd = torch.zeros(2, T - 1, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
            self.acc, self.tok = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, T, dtype=torch.int64, device="cuda")
            self.ws, self.vws = ops.batch_attn_workspace(2, T, P, bt.width * ps, hq, hkv), ops.verify_drafts_workspace(2, T - 1, V)

        def run(self):
            ops.batch_rope_append(self.qkv, cos, sin, self.seq, self.new, self.table, self.k, self.v, hq, hkv, D, self.q)
            ops.batch_attn(self.q, kpre, vpre, kpre.stride(0), P, self.k, self.v, self.table, self.seq, self.new, hq, hkv, D, D ** -0.5, self.out, self.ws)
            ops.verify_drafts(self.logits, self.drafts, self.nd, None, u, 0.9, self.acc, self.tok, self.vws)

        def load(self, i, who):
            r = torch.Generator().manual_seed(100 * i + who)
            self.qkv.copy_((torch.randn(2, T, (hq + 2 * hkv) * D, generator=r)).to(torch.bfloat16))
            self.seq.copy_(torch.randint(0, 61, (2,), generator=r)); self.new.copy_(torch.randint(0, T + 1, (2,), generator=r))
            self.table.copy_(table.flip(0) if i % 2 else table)
            self.logits.copy_(torch.randn(2, T, V, generator=r) * 4)
            self.drafts.copy_(self.logits[:, :T - 1].argmax(-1)); self.nd.copy_(torch.randint(-1, T, (2,), generator=r))

        def state(self):
            return [f64(t) for t in (self.q, self.out, self.k, self.v, self.acc, self.tok)]

    steps, eager = [Step(), Step()], [Step(), Step()]
    for s in steps + eager:
        s.run()                                              # modules loaded before the capture
    torch.cuda.synchronize()
    graphs = []
    for s in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            s.run()
        graphs.append(gr)
    for i in range(4):
        for who in (0, 1):
            steps[who].load(i, who); eager[who].load(i, who)
        for gr in graphs:
            gr.replay()
        for e in eager:
            e.run()
        torch.cuda.synchronize()
        for s, e in zip(steps, eager):
            for a, b in zip(s.state(), e.state()):
                assert np.array_equal(a, b, equal_nan=True)


def test_two_streams_at_once(ops):
    """Two batches in flight on two streams, a workspace each."""
    sets = []
    for seed in (51, 52):
        bt = Batch(4, 16, [30, 400, 4], [1, 1, 1], 1, seed=seed)
        bt.fill([31, 401, 5])
        kpre, vpre = prefix_of(bt, 20_000)
        q = bt.randn(3, 1, 28, D).cuda()
        ws = ops.batch_attn_workspace(3, 1, 20_000, bt.width * 16, 28, 4)
        sets.append((bt, kpre, vpre, q, bt.cuda(), ws, torch.zeros_like(q)))

    def go(s):
        bt, kpre, vpre, q, (kp, vp, table, sl, nn), ws, out = s
        ops.batch_attn(q, kpre, vpre, kpre.stride(0), 20_000, kp, vp, table, sl, nn, 28, 4, D, D ** -0.5, out, ws)

    want = []
    for s in sets:
        go(s)
        torch.cuda.synchronize()
        want.append(s[-1].clone())
        s[-1].zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                go(s)
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert torch.equal(s[-1], w)


# --------------------------------------------------------------------------------------------- every form and shape of the attention, by its size
@pytest.mark.parametrize("hq,hkv,P,ps,seq,T", [
    (2, 1, 8200, 16, [3, 0], 130), (12, 2, 21900, 24, [5], 96), (16, 1, 4100, 16, [7, 0], 512), (4, 4, 16500, 16, [40, 0, 9, 100], 32),
])
def test_attn_prefill_form(ops, hq, hkv, P, ps, seq, T):
    """n_new None and tokens x prefix of two million or more: the prefill kernel, head by head; with the counts given, the same rows by key ranges."""
    bt = Batch(hkv, ps, seq, [T] * len(seq), T, seed=P)
    bt.fill([s + T for s in seq])
    kpre, vpre = prefix_of(bt, P)
    q = bt.randn(bt.B, T, hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=None), ref, tol)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5), ref, tol)


@pytest.mark.parametrize("n_new", ["given", None])
@pytest.mark.parametrize("hq,hkv,P,B,T", [
    (16, 1, 4133, 6, 40), (16, 1, 67001, 8, 12), (28, 4, 17000, 5, 8), (28, 4, 16400, 3, 12), (28, 4, 4000, 20, 1), (28, 4, 16500, 9, 1), (32, 2, 33000, 40, 1),
    (12, 12, 700, 3, 60), (32, 2, 40, 16, 64),
])
def test_attn_many_row_blocks(ops, hq, hkv, P, B, T, n_new):
    """Row blocks of 32, 64, 128 and 256 rows, full, half full and nearly empty; more of them than the card takes at once."""
    rs = np.random.RandomState(P)
    new = rs.randint(0, T + 1, B) if n_new == "given" else np.full(B, T)
    bt = Batch(hkv, 16, rs.randint(0, 40, B).tolist(), new.tolist(), T, seed=B)
    bt.fill([s + n for s, n in zip(bt.seq, bt.new)])
    kpre, vpre = prefix_of(bt, P)
    q = bt.randn(B, T, hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=n_new), ref, tol)


@pytest.mark.parametrize("hq,hkv,P,B,T", [(16, 1, 66000, 3, 6), (16, 1, 66000, 3, 12), (28, 4, 16500, 2, 4), (28, 4, 4000, 8, 12), (16, 1, 4000, 8, 20)])
def test_attn_infinite_values_by_shape(ops, hq, hkv, P, B, T):
    """The prefix's tiles go into LDS unseen; a range that meets a value that is not finite is computed again: in the first, a middle and the last tile."""
    bt = Batch(hkv, 16, [5] * B, [T] * (B - 1) + [T // 2], T, seed=T)
    bt.fill([5 + n for n in bt.new])
    kpre, vpre = prefix_of(bt, P)
    vpre[0, 1, 3] = float("inf"); vpre[0, P // 2, 100] = float("-inf"); vpre[0, P - 1, 7] = float("nan")
    q = bt.randn(B, T, hq, D)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5), ref, tol)


@pytest.mark.parametrize("hq,hkv,P,B,T", [(8, 2, 200, 2, 2), (28, 4, 4000, 3, 1), (28, 4, 16500, 8, 1), (16, 1, 66000, 3, 6), (16, 1, 66000, 3, 12)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attn_a_query_that_is_not_finite_spoils_its_own_rows_only(ops, hq, hkv, P, B, T, value):
    bt = Batch(hkv, 16, [5] * B, [T] * B, T, seed=T)
    bt.fill([5 + T] * B)
    kpre, vpre = prefix_of(bt, P)
    q = bt.randn(B, T, hq, D)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    bad = q.clone()
    bad[B - 1, T - 1, 3, 17] = value
    bad[0, 0, hq - 1] = value
    got = run_attn(ops, bad.cuda(), kpre, vpre, P, bt, hq, D ** -0.5)
    got[B - 1, T - 1, 3], got[0, 0, hq - 1] = 0.0, 0.0                  # (those rows may be anything)
    ref[B - 1, T - 1, 3], ref[0, 0, hq - 1] = 0.0, 0.0
    check(got, ref, tol)


@pytest.mark.parametrize("hq,hkv,P,B,T", [(28, 4, 4000, 20, 1), (28, 4, 20000, 12, 1), (8, 2, 20000, 600, 2), (32, 2, 40000, 48, 1)])
def test_attn_idle_places_may_hold_anything(ops, hq, hkv, P, B, T):
    """Places without a token, in batches that are computed with them: NaN in their queries reaches nothing, their outputs stay as they were."""
    new = [0 if b % 3 else T for b in range(B)]
    bt = Batch(hkv, 16, [b % 7 for b in range(B)], new, T, seed=B)
    bt.fill([s + n for s, n in zip(bt.seq, bt.new)])
    kpre, vpre = prefix_of(bt, P)
    q = torch.full((B, T, hq, D), float("nan"), dtype=torch.bfloat16)
    for b in range(B):
        q[b, :new[b]] = bt.randn(new[b], hq, D)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5), ref, tol)


def test_attn_two_shapes_in_one_workspace_and_captured(ops):
    """A large call and a small one share the larger one's workspace, one behind the other; captured together they replay with other lengths and tokens."""
    hq, hkv, P = 28, 4, 9000
    big, small = Batch(hkv, 16, [30, 0, 9], [20, 7, 20], 20, seed=1), Batch(hkv, 16, [3, 40], [1, 1], 1, seed=2)
    big.fill([52, 22, 31]); small.fill([5, 43])
    kpre, vpre = prefix_of(big, P)
    ws = max((ops.batch_attn_workspace(b.B, b.T, P, b.width * b.ps, hq, hkv) for b in (big, small)), key=lambda t: t.numel())
    calls = []
    for b in (big, small):
        kp, vp, table, sl, nn = b.cuda()
        q = b.randn(b.B, b.T, hq, D)
        calls.append((b, q, q.cuda(), kp, vp, table, sl, nn, torch.full((b.B, b.T, hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")))

    def go():
        for b, _, qd, kp, vp, table, sl, nn, out in calls:
            ops.batch_attn(qd, kpre, vpre, kpre.stride(0), P, kp, vp, table, sl, nn, hq, hkv, D, D ** -0.5, out, ws)

    def compare():
        for b, q, *_, out in calls:
            ref, tol = attn_ref(q, kpre, vpre, P, b, hq, D ** -0.5)
            check(out, ref, tol)

    go(); go()
    torch.cuda.synchronize()
    compare()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
        with torch.cuda.graph(g, stream=s):
            go()
    torch.cuda.current_stream().wait_stream(s)
    for step in range(3):
        big.seq, big.new = [30 + step, step, 9], [20 - step, 7, 1 + step]
        small.seq = [3 + step // 2, 40 + step]
        for (b, q, qd, kp, vp, table, sl, nn, out) in calls:
            sl.copy_(i32(b.seq)); nn.copy_(i32(b.new)); out.fill_(float("nan"))
            q.copy_(b.randn(*q.shape)); qd.copy_(q)
        g.replay()
        torch.cuda.synchronize()
        compare()
        eager = [c[-1].clone() for c in calls]
        go()
        torch.cuda.synchronize()
        for c, e in zip(calls, eager):
            assert np.array_equal(f64(c[-1]), f64(e), equal_nan=True)


def test_attn_infinite_values_in_the_prefill_form(ops):
    hq, hkv, P, T = 4, 2, 8200, 130
    bt = Batch(hkv, 16, [5, 0], [T, T], T, seed=9)
    bt.fill([5 + T, T])
    kpre, vpre = prefix_of(bt, P)
    vpre[0, 0, 3] = float("inf"); vpre[0, P // 2, 5] = float("-inf"); vpre[1, P - 1, 100] = float("-inf"); vpre[1, P - 2, 7] = float("nan")
    q = bt.randn(2, T, hq, D)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=None), ref, tol)


@pytest.mark.parametrize("B,T,n_new", [(12, 1, "given"), (8, 6, "given"), (4, 24, None)])
def test_attn_prefix_heads_past_4_gb(ops, B, T, n_new):
    """Heads of the prefix 2.4 GB apart: the third one's rows lie behind 2^32 bytes, in every form that stages the prefix its own way."""
    hq, hkv, P, stride = 12, 3, 30000, 1_200_000_000
    bt = Batch(hkv, 16, [4] * B, [T] * (B - 1) + [T if n_new is None else 0], T, seed=T)
    bt.fill([4 + n for n in bt.new])
    k, v = bt.randn(hkv, P, D), bt.randn(hkv, P, D)
    far = [torch.empty((hkv - 1) * stride + P * D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    views = [x.as_strided((hkv, P, D), (stride, D, 1)) for x in far]
    views[0].copy_(k); views[1].copy_(v)
    q = bt.randn(B, T, hq, D)
    ref, tol = attn_ref(q, k, v, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), views[0], views[1], P, bt, hq, D ** -0.5, n_new=n_new), ref, tol)


@pytest.mark.parametrize("T,n_new", [(1, "given"), (128, "given"), (128, None)])
def test_attn_probabilities_go_into_the_product_as_two_terms(ops, T, n_new):
    """Two keys have all the weight (the others' e^-350 is 0 in 32 bits), and in column t of row t their values balance: a probability rounded to bf16 once, off by
    up to 2^-8 of it, shows there.  Of two terms 2^-16 is lost; besides that the exponent (products and scores are exact here: 2^-22 max |s|), the exponential
    (2^-21), both again in the normaliser, four fp32 roundings, and the result's own: 2^-8 |o| + (2^-16 + 2 d + 2^-22) sum w |v|.  The same whatever the number
    of tokens, with the counts given and without them."""
    P, scale = 16384, D ** -0.5
    bt = Batch(1, 16, [0], [T], T, seed=3)
    bt.fill([T])
    kpre = torch.zeros(1, P, D, dtype=torch.bfloat16)
    kpre[:, 2:, 1] = -1.0
    kpre[:, 0, 0] = 1.0
    for j in range(T):
        bt.row(bt.k_pool, 0, j).zero_()[:, 1] = -1.0
    q = torch.zeros(1, T, 1, D, dtype=torch.bfloat16)
    q[0, :, 0, 0] = torch.linspace(-9.0, 9.0, T) if T > 1 else 5.0
    q[..., 1] = 4000.0
    s = torch.stack([q[0, :, 0, 0].double() * scale, torch.zeros(T, dtype=torch.float64)], 1)
    vpre = bt.randn(1, P, D)
    vpre[:, 0], vpre[:, 1] = 1.0, 0.5
    vpre[0, 1, :T] = -torch.exp(s[:, 0]).to(torch.bfloat16)
    w = torch.softmax(s, 1)
    ref, size = w @ vpre[0, :2].double(), w @ vpre[0, :2].double().abs()
    d = 2.0 ** -22 * s.abs().amax(1, keepdim=True) + 2.0 ** -21
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -16 + 2 * d + 2.0 ** -22) * size
    got = run_attn(ops, q.cuda(), kpre.cuda(), vpre.cuda(), P, bt, 1, scale, n_new=n_new)
    off = (got[0, :, 0].double().cpu() - ref).abs() - tol
    assert (off <= 0).all(), off.max().item()


# ------------------------------------------------------------------------------------------------------------- values near the type's largest
@pytest.mark.parametrize("hq,hkv,P,B,T,n_new", [(8, 2, 300, 2, 2, "given"), (28, 4, 4000, 3, 1, "given"), (28, 4, 4000, 40, 1, "given"), (28, 4, 4000, 40, 1, None),
                                                (16, 1, 66000, 3, 6, "given"), (28, 4, 16500, 2, 4, "given"), (4, 2, 8200, 2, 130, None)])
def test_attn_large_finite_values_far_below_the_maximum(ops, hq, hkv, P, B, T, n_new):
    """The last half of the prefix scores 360 below its first key (e^-360 is 0 in 32 bits) and holds one finite value row of 1e38: it adds nothing, in whichever
    range it lies; the sequences' own rows score in between and hold one as well."""
    bt = Batch(hkv, 16, [5] * B, [T] * B, T, seed=T)
    bt.fill([5 + T] * B, scale=0.05)
    kpre, vpre = prefix_of(bt, P, scale=0.05)
    kpre[:, 0] = 4.0
    kpre[:, P // 2:P] = -4.0
    vpre[:, P - 2, ::3] = 1.0e38
    for b in range(B):
        bt.row(bt.v_pool, b, 3)[:, 1::3] = -1.0e38
    q = (4.0 + 0.02 * torch.randn(B, T, hq, D, generator=bt.g)).to(torch.bfloat16)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    assert np.isfinite(ref).all() and np.abs(ref).max() < 100
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=n_new), ref, tol)


def test_verify_a_certain_draft_in_a_chunk_that_is_filtered_out(ops):
    """Top-k filters whole chunks of 4096 logits away; the refused draft lies in one of them.  The chunk's sum without the draft is 0, not what the workspace held."""
    B, T, V = 3, 2, 3 * 4096
    x, drafts, _, u = verify_case(B, T, V, torch.float32, False, seed=11)
    x[:, :, 4096:8192] = float("-inf")
    drafts[:] = 5000
    want = verify_ref(x, drafts, None, None, u, 0.8)
    ws = ops.verify_drafts_workspace(B, T, V)
    for stale in (0xff, 0x7f):                                           # NaN; a number of 1e306
        ws.fill_(stale)
        acc, tok = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, T + 1, dtype=torch.int64, device="cuda")
        ops.verify_drafts(x.cuda(), drafts.cuda(), None, None, u.cuda(), 0.8, acc, tok, ws)
        assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
        chunks = 3
        at = (B * (T + 1) * chunks + B * chunks) * 8                     # behind the sums of the rows' chunks and those of the refused rows
        assert ws[at:at + B * T * 8].view(torch.float64).tolist() == [0.0] * (B * T)


@pytest.mark.parametrize("hq,hkv,P,B,T,suffix,n_new", [
    (28, 4, 1000, 64, 1, 20, "given"), (28, 4, 1500, 64, 1, 20, "given"), (28, 4, 700, 73, 1, 40, None), (28, 4, 700, 74, 1, 40, None), (64, 8, 2000, 8, 1, 30, "given"),
    (8, 1, 12000, 16, 1, 9, None), (32, 2, 8000, 2, 1, 700, "given"), (28, 4, 2000, 3, 6, 40, "given"), (28, 4, 2000, 3, 6, 1000, "given"), (28, 4, 900, 4, 4, 5, "given"),
    (33, 1, 700, 3, 1, 100, None), (32, 1, 700, 16, 1, 100, None),
])
@pytest.mark.parametrize("odd", [False, True])
def test_attn_on_both_sides_of_the_one_tile_rule(ops, hq, hkv, P, B, T, suffix, n_new, odd):
    """Batches of up to 512 rows over prefixes of about 256 keys a CU, with few and with many keys of their own, and just beyond; with infinite and NaN values in a
    first, a middle and a last block of 32 keys."""
    rs = np.random.RandomState(P + B)
    new = rs.randint(0, T + 1, B) if n_new == "given" and T > 1 else np.full(B, T)
    bt = Batch(hkv, 16, rs.randint(suffix // 2, suffix + 1, B).tolist(), new.tolist(), T, seed=B)
    bt.fill([s + n for s, n in zip(bt.seq, bt.new)])
    kpre, vpre = prefix_of(bt, P)
    if odd:
        vpre[0, 1, 3] = float("inf"); vpre[0, P // 2, 100] = float("-inf"); vpre[hkv - 1, P - 1, 7] = float("nan")
    q = bt.randn(B, T, hq, D, scale=1.3)
    ref, tol = attn_ref(q, kpre, vpre, P, bt, hq, D ** -0.5)
    check(run_attn(ops, q.cuda(), kpre, vpre, P, bt, hq, D ** -0.5, n_new=n_new), ref, tol)
