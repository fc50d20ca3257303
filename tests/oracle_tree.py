"""Definitions, in 64 bits and row by row, of the operators of a step with trees of drafted tokens, and random steps for their tests."""
import types

import numpy as np
import torch


def line(parents, i):
    """Row i and its ancestors, nearest first; only an earlier row is followed."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def random_parents(rng, n, deep=False):
    """Row 0 is the root; the others follow any earlier row (deep: mostly the one before)."""
    return [-1] + [i - 1 if deep and rng.random() < 0.8 else rng.integers(0, i).item() for i in range(1, n)] if n else []


def bits(parents, words):
    """[n, words] int64 words of rows and their ancestors."""
    out = torch.zeros(len(parents), words, dtype=torch.int64)
    for i in range(len(parents)):
        for j in line(parents, i):
            out[i, j // 64] |= torch.tensor(1 << (j % 64) if j % 64 < 63 else -2 ** 63)
    return out


class Step:
    """Sequences with `before[i]` cached tokens and trees of counts[i] rows over a shuffled cache with garbage in every other place."""

    def __init__(self, before, counts, block, seed=0, words=1, deep=False, spare_rows=0, junk_tables=True):
        rng = np.random.default_rng(seed)
        self.before, self.counts, self.block = before, counts, block
        need = [-(-(b + n) // block) for b, n in zip(before, counts)]
        self.blocks = sum(need) + 1
        MB = max(1, max(need, default=0)) + 2
        ids = (rng.permutation(sum(need)) + 1).tolist()
        # entries behind a sequence's last block are never looked at
        tables = torch.full((len(before), MB), 10 ** 9 if junk_tables else 0, dtype=torch.int32)
        for i, m in enumerate(need):
            for j in range(m):
                tables[i, j] = ids.pop()
        self.parents_of = [random_parents(rng, n, deep) for n in counts]
        T = sum(counts) + spare_rows
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        pos, seq = torch.zeros(T, dtype=torch.int32), torch.full((T,), -1, dtype=torch.int32)
        tree, parents = torch.zeros(T, words, dtype=torch.int64), torch.zeros(T, dtype=torch.int32)
        for i, p in enumerate(self.parents_of):
            a, n = int(cu[i]), counts[i]
            if n:
                parents[a:a + n] = torch.tensor(p)
                tree[a:a + n] = bits(p, words)
                pos[a:a + n] = before[i] + torch.tensor([len(line(p, j)) - 1 for j in range(n)])
                seq[a:a + n] = i
        self.T, self.cu, self.parents = T, cu, parents
        self.inp = types.SimpleNamespace(q_cu=torch.from_numpy(cu), kv_lens=torch.tensor([b + n for b, n in zip(before, counts)], dtype=torch.int32),
                                         block_tables=tables, token_seq=seq, positions=pos, n_seqs=len(before), max_q=max(counts, default=1),
                                         max_kv=max([b + n for b, n in zip(before, counts)], default=0), block_size=block)
        self.tree = tree

    def to(self, device):
        out = types.SimpleNamespace(**vars(self.inp))
        for k, v in vars(self.inp).items():
            if isinstance(v, torch.Tensor):
                setattr(out, k, v.to(device))
        return out

    def place(self, i, p):
        return int(self.inp.block_tables[i, p // self.block]), p % self.block


def attention(q, k_cache, v_cache, step, tree, scale, window=-1):
    """(out, weight) in 64 bits: sum of p v, and sum of p |v| for the bounds of roundings; [T, Hq, D]."""
    T, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    out, size = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    for i, (b, n) in enumerate(zip(step.before, step.counts)):
        if n == 0:
            continue
        where = [step.place(i, p) for p in range(b + n)]
        blk, off = torch.tensor([w[0] for w in where]), torch.tensor([w[1] for w in where])
        k, v = (c[blk, off].double().repeat_interleave(Hq // Hkv, 1) for c in (k_cache, v_cache))
        a = int(step.cu[i])
        pos = step.inp.positions[a:a + n].tolist()
        for r in range(n):
            keys = [j for j in range(b) if window <= 0 or j > pos[r] - window]
            for j in range(min(n, 64 * tree.shape[1])):
                if (int(tree[a + r, j // 64]) >> (j % 64)) & 1 and (window <= 0 or pos[j] > pos[r] - window):
                    keys.append(b + j)
            if not keys:
                continue
            s = torch.einsum("hd,lhd->hl", q[a + r].double(), k[keys]) * scale
            p = torch.softmax(s, -1)
            out[a + r] = torch.einsum("hl,lhd->hd", p, v[keys])
            size[a + r] = torch.einsum("hl,lhd->hd", p, v[keys].abs())
    return out, size


def attention_bound(q, k_cache, out, size, scale, longest, dtype):
    """How far fp32 sums (and bf16 weights and outputs) may take the result from 64 bits.
    Scores: D products and their scaling, each rounded to 2^-24 of at most |q| |k| scale, so every weight is off by a factor e^d; the
    sums over the keys add `longest` such roundings.  bf16: a weight and the output are each rounded by at most 2^-8."""
    D = q.shape[-1]
    most = q.double().norm(dim=-1).max() * k_cache.double().nan_to_num(0, 0, 0).norm(dim=-1).max() * scale
    d = 2.0 ** -24 * (2 * D + 16) * float(most) + 2.0 ** -20
    rel = 2 * d + 2.0 ** -23 * longest
    if dtype == torch.bfloat16:
        return size * (rel + 2.0 ** -8) * (1 + 2.0 ** -7) + out.abs() * 2.0 ** -8 + 1e-30
    return size * rel + out.abs() * 2.0 ** -24 + 1e-30


def logits(x, step_cu, seqs, history, penalties, tokens, parents, bias, mask):
    """(adjusted logits, bound of fp32 roundings), 64 bits."""
    S, V = x.shape
    out, err = x.double().clone(), torch.zeros(S, V, dtype=torch.float64)
    for b in range(len(step_cu) - 1):
        p = b if seqs is None else int(seqs[b])
        a, n = int(step_cu[b]), int(step_cu[b + 1]) - int(step_cu[b])
        pool = history[1].numel() if history is not None else bias[0].numel() - 1 if bias is not None else len(step_cu) - 1
        if not 0 <= p < pool:
            continue
        up = [int(v) for v in parents[a:a + n]] if parents is not None else list(range(-1, n - 1))
        for r in range(n):
            if history is not None:
                ids = [int(v) for v in history[0][p, :int(history[1][p])]]
                made = ids[int(history[2][p]):]
                if tokens is not None:
                    mine = [int(tokens[a + j]) for j in reversed(line(up, r))]
                    ids, made = ids + mine, made + [t for j, t in enumerate(mine) if int(history[1][p]) + j >= int(history[2][p])]
                rep, freq, pres = (float(t[p]) for t in penalties)
                for i in set(ids):
                    if 0 <= i < V:
                        c = made.count(i)
                        y = out[a + r, i] - c * freq - (pres if c else 0.0)
                        big = abs(float(out[a + r, i])) + c * abs(freq) + abs(pres)
                        out[a + r, i] = y * rep if y < 0 else y / rep
                        err[a + r, i] = 2.0 ** -24 * 5 * big * max(rep, 1 / rep)
            if bias is not None:
                add = {int(bias[1][e]): float(bias[2][e]) for e in range(int(bias[0][p]), int(bias[0][p + 1]))}
                for i, v in add.items():
                    if 0 <= i < V:
                        out[a + r, i] += v
                        err[a + r, i] += 2.0 ** -24 * (abs(float(out[a + r, i])) + abs(v))
    if mask is not None:
        for r in range(S):
            m = int(mask[1][r])
            if 0 <= m < mask[0].shape[0]:
                for i in range(V):
                    if not (int(mask[0][m, i // 32]) >> (i % 32)) & 1:
                        out[r, i] = -float("inf")
                        err[r, i] = 0
    return out, err


def accepted_path(tokens, parents, target, depth):
    rows = [0] if len(tokens) else []
    while rows and len(rows) <= depth:
        nxt = [j for j in range(rows[-1] + 1, len(tokens)) if parents[j] == rows[-1] and tokens[j] == target[rows[-1]]]
        if not nxt:
            break
        rows.append(nxt[0])
    return rows
