"""CPU doubles of the batch operators (plain torch, fp32) on top of tests/oracle_ops.py, so that the host logic of quickvideo_amd/batch.py - pages,
forks, lengths, drafts - runs in the CPU suite."""
import torch
from oracle_ops import OracleOps


class BatchOracleOps(OracleOps):
    @staticmethod
    def _counts(n_new, B, T):
        return [T] * B if n_new is None else [max(0, min(T, int(n))) for n in n_new.tolist()]

    def batch_rope_append(self, qkv, cos, sin, seq_len, n_new, table, k_pages, v_pages, n_q, n_kv, D, q_out):
        B, T = qkv.shape[:2]
        ps = k_pages.shape[2]
        x = qkv.view(B, T, n_q + 2 * n_kv, D).float()
        c, s = cos.view(B, T, 1, D // 2).float(), sin.view(B, T, 1, D // 2).float()
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(torch.bfloat16)
        for b, n in enumerate(self._counts(n_new, B, T)):
            for t in range(n):
                j = int(seq_len[b]) + t
                page = int(table[b, j // ps])
                assert 0 <= page < k_pages.shape[0], "a row without a page"
                q_out[b, t] = y[b, t, :n_q]
                k_pages[page, :, j % ps] = y[b, t, n_q:n_q + n_kv]
                v_pages[page, :, j % ps] = x[b, t, n_q + n_kv:].to(torch.bfloat16)

    def batch_attn(self, q, k_prefix, v_prefix, stride, P, k_pages, v_pages, table, seq_len, n_new, n_q, n_kv, D, scale, out, ws):
        B, T = q.shape[:2]
        ps, G = k_pages.shape[2], n_q // n_kv
        for b, n in enumerate(self._counts(n_new, B, T)):
            for t in range(n):
                m = int(seq_len[b]) + t + 1
                pages = table[b, :-(-m // ps)].long()
                for h in range(n_kv):
                    k = torch.cat([k_prefix[h, :P], k_pages[pages, h].reshape(-1, D)[:m]]).float()
                    v = torch.cat([v_prefix[h, :P], v_pages[pages, h].reshape(-1, D)[:m]]).float()
                    w = torch.softmax(q[b, t, h * G:(h + 1) * G].float() @ k.t() * scale, -1)
                    out[b, t, h * G:(h + 1) * G] = (w @ v).to(torch.bfloat16)

    def verify_drafts(self, logits, drafts, n_draft, draft_probs, uniforms, temperature, n_accepted, tokens, ws):
        assert draft_probs is None
        tokens.fill_(-1)
        for b in range(logits.shape[0]):
            n, T = int(n_draft[b]), logits.shape[1] - 1
            for a in range(n + 1):
                x = logits[b, a].double()
                d = int(drafts[b, a]) if a < n else -1
                if temperature == 0:
                    nxt = int(x.argmax())
                    stands = d == nxt
                else:
                    p = torch.softmax(x / temperature, -1)
                    stands = a < n and float(uniforms[b, a]) < float(p[d])
                    if a < n:
                        p[d] = 0
                    run = p.cumsum(0)
                    nxt = int(((run > float(uniforms[b, T]) * run[-1]) & (p > 0)).long().argmax())
                if a < n and stands:
                    tokens[b, a] = d
                    continue
                tokens[b, a] = nxt
                n_accepted[b] = a
                break
