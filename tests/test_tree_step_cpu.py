"""Steps with trees of drafted tokens on the CPU: the operators against their definitions, what they refuse, and a whole model that
verifies trees and goes on exactly as without them."""
import types

import numpy as np
import pytest
import torch

import oracle_tree as oracle
from xllm_wxh_b200 import ops
from xllm_wxh_b200.framework.step_input import TreeStep

I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32)


# ----------------------------------------------------------------------------- step_rows
@pytest.mark.parametrize("block", [1, 4, 16])
def test_step_rows_chain_and_padding(block):
    tables = torch.arange(1, 5 * 40 + 1, dtype=I32).view(5, 40)
    lens = ints(0, 3, 15, 16, 17)
    r = ops.step_rows(tables, lens, ints(4, -1, 0, 2, 9), ints(2, 5, 1, 3, 4), 10, block)
    assert r.q_cu.tolist() == [0, 2, 2, 3, 6, 6] and r.kv_lens.tolist() == [19, 0, 1, 18, 0] and r.tree is None
    assert r.positions.tolist() == [17, 18, 0, 15, 16, 17, 0, 0, 0, 0]
    assert r.token_seq.tolist() == [0, 0, 2, 3, 3, 3, -1, -1, -1, -1]
    want = [int(tables[s, p // block]) * block + p % block for s, p in [(4, 17), (4, 18), (0, 0), (2, 15), (2, 16), (2, 17)]]
    assert r.slots.tolist() == want + [t % block for t in range(6, 10)]
    used = [-(-k // block) for k in r.kv_lens.tolist()]
    for b, s in enumerate([4, -1, 0, 2, -1]):
        assert r.block_tables[b].tolist() == (tables[s, :used[b]].tolist() if s >= 0 else []) + [0] * (40 - used[b])


def test_step_rows_trees():
    rng = np.random.default_rng(1)
    counts = [1, 70, 0, 8]
    ps = [oracle.random_parents(rng, n) for n in counts]
    ps[3] = [-1, 0, 0, 1, 3, 7, -9, 4]                    # a row that names itself or a later one, or nothing, follows the cached tokens
    tables = torch.randint(1, 1000, (4, 9), dtype=I32)
    parents = torch.tensor([v for p in ps for v in p] + [0], dtype=I32)
    r = ops.step_rows(tables, ints(5, 0, 7, 60), ints(0, 1, 2, 3), torch.tensor(counts, dtype=I32), 80, 16, parents, max_q=70, max_blocks=6)
    assert r.block_tables.shape == (4, 6)
    at = 0
    for b, (p, before) in enumerate(zip(ps, [5, 0, 7, 60])):
        for i in range(len(p)):
            up = oracle.line(p, i)
            assert int(r.positions[at + i]) == before + len(up) - 1
            assert torch.equal(r.tree[at + i], oracle.bits(p, 2)[i])
        at += len(p)
    assert r.tree[79].tolist() == [0, 0]


def test_step_rows_refusals():
    tables, lens, one = torch.ones(2, 4, dtype=I32), ints(1, 2), ints(1, 1)
    ok = dict(tables=tables, lens=lens, seqs=ints(0, 1), counts=one, n_rows=2, block_size=4)
    ops.step_rows(**ok)
    for bad in [dict(tables=tables.long()), dict(lens=ints(1)), dict(lens=lens.float()), dict(seqs=ints(0)), dict(counts=one.long()), dict(n_rows=-1),
                dict(block_size=0), dict(max_blocks=5), dict(parents=ints(0)), dict(parents=torch.zeros(300, dtype=I32), n_rows=300),
                dict(max_q=0), dict(tables=tables.t())]:
        with pytest.raises(AssertionError):
            ops.step_rows(**{**ok, **bad})


# ----------------------------------------------------------------------------- attention
def attention_inputs(step, Hq, Hkv, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(step.T, Hq, D, generator=g).to(dtype)
    caches = [torch.randn(step.blocks, step.block, Hkv, D, generator=g).to(dtype) for _ in range(2)]
    return q, *caches


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("before,counts,block,window", [([0], [1], 4, -1), ([5, 0, 33], [7, 3, 12], 8, -1), ([40, 9], [6, 70], 16, 11), ([3, 8], [0, 5], 1, 2)])
def test_tree_attention(before, counts, block, window, dtype):
    step = oracle.Step(before, counts, block, seed=2, words=2, spare_rows=2, junk_tables=False)
    q, k, v = attention_inputs(step, 6, 2, 24, dtype)
    got = ops.tree_attention(q, k, v, step.inp, step.tree, 0.3, window).view(step.T, 6, 24)
    want, size = oracle.attention(q, k, v, step, step.tree, 0.3, window)
    assert ((got.double() - want).abs() <= oracle.attention_bound(q, k, want, size, 0.3, 200, dtype)).all()
    assert not got[sum(counts):].any()


def test_tree_attention_masks_of_any_kind():
    step = oracle.Step([0, 4], [5, 6], 4, seed=3)
    q, k, v = attention_inputs(step, 2, 1, 8, torch.float32)
    tree = torch.randint(-2 ** 62, 2 ** 62, step.tree.shape)
    tree[1] = 0                                            # sees nothing at all
    tree[5] = 0                                            # sees the cached tokens only
    got = ops.tree_attention(q, k, v, step.inp, tree, 1.0).view(-1, 2, 8)
    want, size = oracle.attention(q, k, v, step, tree, 1.0)
    assert not got[1].any() and ((got.double() - want).abs() <= oracle.attention_bound(q, k, want, size, 1.0, 16, q.dtype)).all()


def test_tree_attention_refusals():
    step = oracle.Step([4], [3], 4, junk_tables=False)
    q, k, v = attention_inputs(step, 4, 2, 8, torch.float32)
    ok = dict(q=q, k_cache=k, v_cache=v, inp=step.inp, tree=step.tree, scale=1.0)
    ops.tree_attention(**ok)
    other = lambda **kw: types.SimpleNamespace(**{**vars(step.inp), **kw})
    for bad in [dict(q=q.half(), k_cache=k.half(), v_cache=v.half()), dict(q=q.bfloat16()), dict(v_cache=v[..., :4].contiguous()), dict(q=q[:, :3]),
                dict(k_cache=k.transpose(1, 2)), dict(tree=step.tree.int()), dict(tree=step.tree[:2]), dict(tree=torch.zeros(3, 5, dtype=torch.int64)),
                dict(inp=other(q_cu=step.inp.q_cu.long())), dict(inp=other(kv_lens=ints(1, 2))), dict(inp=other(positions=ints(1)))]:
        with pytest.raises(AssertionError):
            ops.tree_attention(**{**ok, **bad})


def test_other_attention_refuses_trees():
    inp = types.SimpleNamespace(tree=torch.zeros(1, 1, dtype=torch.int64))
    with pytest.raises(NotImplementedError):
        ops.paged_attention_ext(None, None, None, inp, 1.0)
    with pytest.raises(NotImplementedError):
        ops.mla_attention(None, None, None, inp, 1.0, 512)
    with pytest.raises(NotImplementedError):
        ops.latent_attention(torch.zeros(1, 2, 24), torch.zeros(2, 8, 16), torch.zeros(2, 16, 8), torch.zeros(1, 4, 16), inp, None, 1.0, 16)


# ----------------------------------------------------------------------------- logits
def rules(V, pool, rows_of, seed, dtype=torch.float32, masked=True, tree=True):
    """Random histories, penalties, tokens, biases (some ids twice) and masks for `rows_of[b]` rows per sequence."""
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    S, B = sum(rows_of), len(rows_of)
    r = types.SimpleNamespace(V=V, cu=torch.tensor(np.concatenate([[0], np.cumsum(rows_of)]), dtype=I32), seqs=torch.from_numpy(rng.permutation(pool)[:B].astype(np.int32)))
    r.logits = (torch.randn(S, V, generator=g) * 4).to(dtype)
    cap = 37
    lens = torch.randint(0, cap + 1, (pool,), generator=g, dtype=I32)
    prompts = (lens * torch.rand(pool, generator=g)).int()
    prompts[::2] = lens[::2] + 1                           # the rows begin with the prompt's last token
    r.history = (torch.randint(0, max(1, V // 2), (pool, cap), generator=g, dtype=I32), lens, prompts)
    r.penalties = (torch.rand(pool, generator=g) + 0.5, torch.rand(pool, generator=g) - 0.3, torch.rand(pool, generator=g) - 0.3)
    r.tokens = torch.randint(0, V, (S,), generator=g, dtype=I32)
    r.parents = torch.tensor([v for n in rows_of for v in oracle.random_parents(rng, n)], dtype=I32) if tree else None
    n = torch.randint(0, 6, (pool,), generator=g)
    cu = torch.zeros(pool + 1, dtype=I32)
    cu[1:] = n.cumsum(0)
    r.bias = (cu, torch.randint(0, max(1, V // 8), (int(cu[-1]),), generator=g, dtype=I32), torch.randn(int(cu[-1]), generator=g) * 3)
    r.mask = None
    if masked:
        words = torch.randint(-2 ** 31, 2 ** 31, (S, -(-V // 32)), generator=g, dtype=torch.int64).int()
        words[0] = -1
        words[-1] = 0
        r.mask = (words, torch.from_numpy(rng.integers(-1, S, S).astype(np.int32)))
    return r


def check_rules(r, got, dtype):
    want, err = oracle.logits(r.logits, r.cu, r.seqs, r.history, r.penalties, r.tokens, r.parents, r.bias, r.mask)
    if dtype == torch.bfloat16:
        err = err * 1.01 + torch.where(want.isfinite(), want.abs(), torch.zeros_like(want)) * 2.0 ** -8
    inf = want == -float("inf")
    assert torch.equal(inf, got.double() == -float("inf"))
    assert ((got.double() - want).masked_fill(inf, 0).abs() <= err.masked_fill(inf, 0)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,rows_of,masked,tree", [(50, [1, 1, 1], True, False), (97, [4, 0, 9], True, True), (64, [3], False, True)])
def test_adjust_logits(V, rows_of, masked, tree, dtype):
    r = rules(V, len(rows_of) + 2, rows_of, 5, dtype, masked, tree)
    got = r.logits.clone()
    assert ops.adjust_logits(got, r.cu, r.seqs, r.history, r.penalties, r.tokens, r.parents, r.bias, r.mask) is got
    check_rules(r, got, dtype)


def test_adjust_logits_agrees_with_the_penalties_of_sample():
    """Histories without drafted rows: the same penalties as (id, count) lists."""
    from xllm_wxh_b200.ops import reference as ref
    r = rules(40, 3, [1, 1, 1], 9, masked=False, tree=False)
    r.seqs = ints(0, 1, 2)
    got = ops.adjust_logits(r.logits.clone(), r.cu, None, r.history, r.penalties)
    cu, ids, counts = [0], [], []
    for p in range(3):
        text = r.history[0][p, :int(r.history[1][p])].tolist()
        made = text[int(r.history[2][p]):]
        for i in sorted(set(text)):
            ids.append(i)
            counts.append(text.count(i) | made.count(i) << 16)
        cu.append(len(ids))
    want = ref.apply_penalties(r.logits.clone(), ints(*cu), ints(*ids), ints(*counts), *r.penalties)
    assert torch.allclose(got, want, rtol=2e-6, atol=1e-6)


def test_adjust_logits_refusals():
    r = rules(40, 3, [2, 1, 1], 4)
    ok = dict(logits=r.logits, q_cu=r.cu, seqs=r.seqs, history=r.history, penalties=r.penalties, tokens=r.tokens, parents=r.parents, bias=r.bias, mask=r.mask)
    for bad in [dict(logits=r.logits.half()), dict(logits=r.logits.t()), dict(q_cu=r.cu.long()), dict(seqs=r.seqs[:1]), dict(penalties=None),
                dict(penalties=r.penalties[:2]), dict(history=None), dict(tokens=None), dict(tokens=r.tokens[:1]), dict(parents=r.parents.long()),
                dict(bias=(r.bias[0][:2], *r.bias[1:])), dict(bias=(*r.bias[:2], r.bias[2].double())), dict(mask=(r.mask[0][:, :1], r.mask[1])),
                dict(mask=(r.mask[0], r.mask[1][:1])), dict(max_q=257), dict(max_q=0), dict(history=(r.history[0].long(), *r.history[1:]))]:
        with pytest.raises(AssertionError):
            ops.adjust_logits(**{**ok, **bad})


# ----------------------------------------------------------------------------- accept_tree
def acceptance(step, seed, vocab=3):
    rng = np.random.default_rng(seed)
    step.inp.tokens = torch.from_numpy(rng.integers(0, vocab, step.T).astype(np.int32))       # few ids: siblings with the same token
    return torch.from_numpy(rng.integers(0, vocab, step.T).astype(np.int32))


def expected_acceptance(step, target, caches, depth):
    out = [c.clone() for c in caches]
    rows_of = []
    for i, n in enumerate(step.counts):
        a = int(step.cu[i])
        rows = oracle.accepted_path(step.inp.tokens[a:a + n].tolist(), step.parents_of[i], target[a:a + n].tolist(), depth)
        rows_of.append((a, rows))
        for j, r in enumerate(rows):
            (b0, o0), (b1, o1) = step.place(i, step.before[i] + r), step.place(i, step.before[i] + j)
            for o, c in zip(out, caches):
                o[b1, o1] = c[b0, o0]
    return rows_of, out


def check_acceptance(step, target, result, depth, rows_of):
    out, accepted, path = (t.tolist() for t in result)
    for i, (a, rows) in enumerate(rows_of):
        pad = [-1] * (depth + 1 - len(rows))
        assert out[i] == [int(target[a + r]) for r in rows] + pad and path[i] == rows + pad and accepted[i] == max(len(rows) - 1, 0)


@pytest.mark.parametrize("before,counts,block,depth", [([0], [1], 4, 0), ([5, 0, 30], [9, 0, 40], 4, 12), ([7, 7], [12, 64], 16, 63), ([2], [30], 8, 2)])
def test_accept_tree(before, counts, block, depth):
    step = oracle.Step(before, counts, block, seed=6, deep=True)
    target = acceptance(step, 7)
    caches = [torch.randn(step.blocks, block, 3, 4), torch.randint(0, 100, (step.blocks, block, 5))]
    rows_of, want = expected_acceptance(step, target, caches, depth)
    result = ops.accept_tree(target, step.inp, step.parents, caches, depth)
    check_acceptance(step, target, result, depth, rows_of)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_accept_tree_refusals():
    step = oracle.Step([4], [3], 4)
    target = acceptance(step, 1)
    cache = torch.zeros(step.blocks, 4, 2)
    ok = dict(target=target, inp=step.inp, parents=step.parents, caches=[cache])
    ops.accept_tree(**ok)
    for bad in [dict(target=target.long()), dict(parents=step.parents[:2]), dict(caches=[cache, cache]), dict(caches=[cache.transpose(0, 1)]),
                dict(caches=[torch.zeros(step.blocks, 8, 2)]), dict(max_depth=-1), dict(max_depth=256),
                dict(inp=types.SimpleNamespace(**{**vars(step.inp), "max_q": 300}))]:
        with pytest.raises(AssertionError):
            ops.accept_tree(**{**ok, **bad})


def test_accept_tree_refuses_caches_that_overlap():
    step = oracle.Step([4], [3], 4)
    n = step.blocks
    both = torch.zeros(2 * n, 4, 2)
    with pytest.raises(AssertionError):
        ops.accept_tree(acceptance(step, 1), step.inp, step.parents, [both[:n], both[n - 1:]])
    ops.accept_tree(acceptance(step, 1), step.inp, step.parents, [both[:n], both[n:]])


# ----------------------------------------------------------------------------- together
def test_tree_step_needs_trees():
    r = ops.step_rows(torch.ones(1, 4, dtype=I32), ints(0), ints(0), ints(2), 2, 4)
    with pytest.raises(ValueError):
        TreeStep(ints(1, 2), r, 4, 2, 2)


def test_model_goes_on_as_without_drafts():
    from helpers.tree_generation import check_generation
    check_generation("cpu", torch.float32)
