"""Kernels of a step with trees of drafted tokens at the edges of what their documentation allows: empty histories, tables and caches,
positions of any kind, values that are not finite, vocabularies of several slices."""
import types

import pytest
import torch

import oracle_tree as oracle
from test_tree_step_cpu import acceptance, attention_inputs, check_rules, rules
from test_tree_step_gpu import check_attention, cuda, status      # noqa: F401 (every test reads the status word)
from xllm_wxh_b200 import ops

pytestmark = pytest.mark.gpu
I32 = torch.int32

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adjust_logits_history_without_columns(dtype):
    """Histories that hold nothing yet: the rows' own tokens are penalised all the same."""
    r = rules(200, 5, [4, 1, 7], 11, dtype)
    r.history = (r.history[0][:, :0], torch.zeros_like(r.history[1]), torch.zeros_like(r.history[2]))
    got = r.logits.cuda()
    ops.adjust_logits(got, *cuda((r.cu, r.seqs, r.history, r.penalties, r.tokens, r.parents, r.bias, r.mask)), max_q=7)
    check_rules(r, got.cpu(), dtype)
    # a pool without requests: every sequence lies outside
    none = ((r.history[0][:0], r.history[1][:0], r.history[2][:0]), tuple(p[:0] for p in r.penalties))
    got = r.logits.cuda()
    ops.adjust_logits(got, *cuda((r.cu, r.seqs, *none, r.tokens, r.parents)), max_q=7)
    assert torch.equal(got.cpu(), r.logits)

@pytest.mark.parametrize("window", [1, 40, 150])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float32)])
def test_tree_attention_window_with_positions_of_any_kind(window, D, dtype):
    """A row's position counts as one of its sequence's rows': the nearest one."""
    step = oracle.Step([0, 5, 64, 200, 700], [9, 30, 3, 64, 12], 16, seed=4, deep=True)
    q, k, v = attention_inputs(step, 8, 2, D, dtype)
    given = step.inp.positions + torch.randint(-400, 400, (step.T,), generator=torch.Generator().manual_seed(window), dtype=I32)
    given[3], given[50] = 2 ** 31 - 1, -2 ** 31
    first = torch.repeat_interleave(torch.tensor(step.before), torch.tensor(step.counts)).int()
    last = first + torch.repeat_interleave(torch.tensor(step.counts), torch.tensor(step.counts)).int() - 1
    step.inp.positions = given
    inp = step.to("cuda")
    step.inp.positions = given.clamp(first, last)
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), inp, step.tree.cuda(), D ** -0.5, window).view(step.T, 8, D).cpu().double()
    want, size = oracle.attention(q, k, v, step, step.tree, D ** -0.5, window)
    assert ((got - want).abs() <= oracle.attention_bound(q, k, want, size, D ** -0.5, 712, dtype)).all()

@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (64, torch.float32), (192, torch.bfloat16)])
def test_tree_attention_without_table_columns_or_blocks(D, dtype):
    """No place to read from: every row sees nothing."""
    step = oracle.Step([20, 5], [6, 4], 16, seed=3, spare_rows=2)
    q, k, v = attention_inputs(step, 4, 2, D, dtype)
    inp = step.to("cuda")
    inp.block_tables = inp.block_tables[:, :0].contiguous()
    assert not ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), inp, step.tree.cuda(), 0.3).any()
    inp.block_tables, inp.kv_lens = step.inp.block_tables.cuda(), torch.zeros_like(inp.kv_lens)
    assert not ops.tree_attention(q.cuda(), k[:0].cuda(), v[:0].cuda(), inp, step.tree.cuda(), 0.3).any()
    none = types.SimpleNamespace(**{**vars(inp), "positions": inp.positions[:0], "token_seq": inp.token_seq[:0], "q_cu": torch.zeros_like(inp.q_cu),
                                    "block_tables": inp.block_tables[:, :0].contiguous()})
    assert ops.tree_attention(q[:0].cuda(), k.cuda(), v.cuda(), none, step.tree[:0].cuda(), 0.3).shape == (0, 4 * D)


def test_tree_attention_refuses_heads_and_blocks_of_nothing():
    step = oracle.Step([4], [3], 16)
    q, k, v = (t.cuda() for t in attention_inputs(step, 4, 2, 64, torch.bfloat16))
    inp, tree = step.to("cuda"), step.tree.cuda()
    for bad in [dict(q=q[:, :0]), dict(q=q[..., :0], k=k[..., :0], v=v[..., :0]), dict(k=k[:, :, :0], v=v[:, :, :0]), dict(k=k[:, :0], v=v[:, :0])]:
        a = {**dict(q=q, k=k, v=v), **bad}
        with pytest.raises(AssertionError):
            ops.tree_attention(a["q"], a["k"], a["v"], inp, tree, 1.0)

def test_tree_attention_tables_of_more_places_than_32_bits_count():
    """Tables so wide that their key tiles, over all sequences and heads, pass 2^31."""
    step = oracle.Step([300, 0, 41, 7, 100, 64, 65, 1], [5, 1, 9, 0, 3, 2, 2, 16], 8192, seed=3)
    q, k, v = attention_inputs(step, 16, 8, 8, torch.bfloat16)
    inp = step.to("cuda")
    inp.block_tables = torch.zeros(8, 2 ** 19, dtype=I32, device="cuda")
    inp.block_tables[:, 0] = step.inp.block_tables[:, 0].cuda() % step.blocks
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), inp, step.tree.cuda(), 0.3).view(step.T, 16, 8).cpu().double()
    want, size = oracle.attention(q, k, v, step, step.tree, 0.3)
    assert ((got - want).abs() <= oracle.attention_bound(q, k, want, size, 0.3, 305, torch.bfloat16)).all()

def check_not_finite(step, q, k, v, dtype, scale=1.0):
    """Numbers come out where the definition has numbers, and nowhere else."""
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), scale).view(q.shape).cpu().double()
    want, size = oracle.attention(q, k, v, step, step.tree, scale)
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite())
    longest = max(b + n for b, n in zip(step.before, step.counts))
    off = (got - want).abs() - oracle.attention_bound(q, k, want, size, scale, longest, dtype)
    assert not (off[fine] > 0).any()
    return fine


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("before,at", [(2000, 5), (2000, 1998), (2000, 2001), (20, 5), (20, 21)])
def test_tree_attention_visible_values_and_scores_that_are_not_finite(before, at, bad, dtype):
    """A row whose scores are not all numbers, or that sees a value that is not finite, does not become finite because other keys outweigh
    that one by more than fp32 holds."""
    step = oracle.Step([before], [3], 16, seed=5)
    step.tree[:] = 7                                             # every row sees all three
    q, k, v = attention_inputs(step, 2, 1, 64, dtype)
    q.fill_(1)
    k.mul_(0.125)
    for p in range(at // 64 * 64, min(at // 64 * 64 + 64, before + 3)):
        k[step.place(0, p)] = -10                                # scores of -640 among keys whose scores are about 0
    if before < 64:
        k[step.place(0, 1)] = 0.5                                # one score of 32 among them
    v[step.place(0, at)][..., 9] = bad
    fine = check_not_finite(step, q, k, v, dtype)
    assert not fine[..., 9].any() and fine[..., :9].all()
    v[step.place(0, at)][..., 9] = 1
    k[step.place(0, at)][..., 4] = float("nan")
    assert not check_not_finite(step, q, k, v, dtype).any()

def seen_bound(step, q, k, want, size, scale, longest, dtype, hidden):
    """The bound of roundings from the keys that some row sees."""
    k = k.clone()
    k[hidden] = 0
    return oracle.attention_bound(q, k, want, size, scale, longest, dtype)


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float32), (192, torch.bfloat16)])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("before,n,window", [(70, 10, -1), (3, 70, -1), (300, 12, 50), (128, 4, -1), (60, 3, -1), (900, 20, 100)])
def test_tree_attention_largest_numbers_behind_masks(before, n, window, sign, D, dtype):
    """The largest finite numbers in places that no row sees, and in branches that others see: bounds by what a row sees."""
    step = oracle.Step([before, 9], [n, 2], 16, seed=7, words=2)
    q, k, v = attention_inputs(step, 8, 2, D, dtype)
    hidden = torch.ones(step.blocks, step.block, dtype=torch.bool)
    for i, (b, m) in enumerate(zip(step.before, step.counts)):
        for p in range(max(0, b - window) if window > 0 else 0, b + m):
            hidden[step.place(i, p)] = False
    k[hidden], v[hidden] = sign * torch.finfo(dtype).max, sign * torch.finfo(dtype).max
    scale = D ** -0.5
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), scale, window).view(step.T, 8, D).cpu().double()
    want, size = oracle.attention(q, k, v, step, step.tree, scale, window)
    bound = seen_bound(step, q, k, want, size, scale, before + n, dtype, hidden)
    # a weight's and the result's roundings, 2^-8 each, of values below 8: far below the values themselves
    assert bound.max() < 0.07 and want.abs().max() > 1
    assert ((got - want).abs() <= bound).all()
    # the last row, which no other sees, holds the largest numbers as values and keys: the other rows are as before
    last = int(step.cu[1]) - 1
    k[step.place(0, before + n - 1)], v[step.place(0, before + n - 1)] = -sign * torch.finfo(dtype).max, sign * torch.finfo(dtype).max
    rest = torch.arange(step.T) != last
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), scale, window).view(step.T, 8, D).cpu().double()
    assert ((got - want).abs() <= bound)[rest].all()

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,length", [(262149, 40), (262213, 20000), (600000, 300)])
def test_adjust_logits_vocabulary_of_several_slices(V, length, dtype):
    """More ids than a bitmap holds: histories, paths, biases and masks on either side of the border between slices."""
    g = torch.Generator().manual_seed(length)
    edge = torch.tensor([0, 31, 262142, 262143, 262144, 262145, V - 1], dtype=I32)
    ids = torch.randint(0, V, (3, length), generator=g, dtype=I32)
    ids[:, :14] = edge.repeat(2)
    ids[1] = ids[1, :14].repeat(length // 14 + 1)[:length]
    lens, prompts = torch.tensor([length, length - 1, 3], dtype=I32), torch.tensor([length // 2, 0, 9], dtype=I32)
    pen = (torch.tensor([1.3, 0.7, 1.5]), torch.tensor([0.1, -0.02, 0.3]), torch.tensor([0.5, 0.1, 0.0]))
    cu, seqs = torch.tensor([0, 3, 4, 6], dtype=I32), torch.tensor([2, 0, 1], dtype=I32)
    tokens = torch.tensor([262143, 262144, V - 1, 262144, 5, 262143], dtype=I32)
    parents = torch.tensor([-1, 0, 1, -1, -1, 0], dtype=I32)
    n = 50
    bias = (torch.tensor([0, n, 2 * n, 3 * n], dtype=I32), torch.randint(0, V, (3 * n,), generator=g, dtype=I32), torch.randn(3 * n, generator=g))
    bias[1][:7], bias[1][n:n + 7] = edge, edge.flip(0)
    bias[1][7] = 262144                                           # twice: the last one holds
    words = torch.randint(-2 ** 31, 2 ** 31, (2, -(-V // 32)), generator=g, dtype=torch.int64).int()
    words[0, 262112 // 32:262176 // 32] = -1
    of = torch.tensor([0, 1, -1, 0, 0, -1], dtype=I32)
    x = (torch.randn(6, V, generator=g) * 3).to(dtype)
    got = x.cuda()
    ops.adjust_logits(got, *cuda((cu, seqs, (ids, lens, prompts), pen, tokens, parents, bias, (words, of))), max_q=3)
    got = got.cpu().double()
    allowed = ((words[..., None] >> torch.arange(32).int()) & 1).flatten(1)[:, :V].bool()
    for b, p in enumerate(seqs.tolist()):
        text = ids[p, :int(lens[p])].long()
        seen, made = torch.bincount(text, minlength=V), torch.bincount(text[int(prompts[p]):], minlength=V)
        add = torch.zeros(V, dtype=torch.float64)
        for i, v in zip(bias[1][p * n:(p + 1) * n].tolist(), bias[2][p * n:(p + 1) * n].tolist()):
            add[i] = v
        rep, freq, pres = (float(t[p].double()) for t in pen)
        for r in range(int(cu[b]), int(cu[b + 1])):
            a = int(cu[b])
            mine = [int(tokens[a + j]) for j in reversed(oracle.line(parents[a:int(cu[b + 1])].tolist(), r - a))]
            behind = [t for j, t in enumerate(mine) if int(lens[p]) + j >= int(prompts[p])]
            count = lambda t: torch.bincount(torch.tensor(t, dtype=torch.int64), minlength=V)
            c = (made + count(behind)).double()
            y = x[r].double()
            z = y - c * freq - (c > 0) * pres
            z = torch.where(seen + count(mine) > 0, torch.where(z < 0, z * rep, z / rep), y) + add
            # six roundings of fp32 to values of at most this size
            big = (y.abs() + c * abs(freq) + abs(pres)) * max(rep, 1 / rep) + add.abs()
            bound = 2.0 ** -24 * 6 * big + (z.abs() * 2.0 ** -8 * 1.01 if dtype == torch.bfloat16 else 0)
            open_ = allowed[of[r]] if of[r] >= 0 else torch.ones(V, dtype=torch.bool)
            assert (got[r][~open_] == -float("inf")).all()
            assert ((got[r] - z).abs() <= bound)[open_].all()

def test_adjust_logits_refuses_parts_that_are_missing():
    f, i = torch.ones(1, device="cuda"), lambda *v: torch.tensor(v, dtype=I32).cuda()
    x, words = torch.zeros(3, 40, device="cuda"), torch.zeros(1, 2, dtype=I32, device="cuda")
    ok = dict(logits=x, q_cu=i(0, 3), history=(i(1, 2).view(1, 2), i(2), i(1)), penalties=(f, f, f), mask=(words, i(-1, -1, -1)), bias=(i(0, 1), i(4), f))
    for name in ("history", "penalties", "mask", "bias"):
        for missing in range(len(ok[name])):
            part = tuple(None if j == missing else t for j, t in enumerate(ok[name]))
            with pytest.raises(AssertionError):
                ops.adjust_logits(**{**ok, name: part})
    assert not x.any()
    ops.adjust_logits(**ok)

def test_accept_tree_places_outside_tables_and_caches():
    """Tables too short for the path, entries that name no block, fewer keys than rows, caches of different lengths: those rows stay."""
    step = oracle.Step([6, 9, 0], [20, 12, 9], 4, seed=6, deep=True, junk_tables=False)
    target = acceptance(step, 7, 1)
    for a, n in zip(step.cu.tolist(), step.counts):              # two rows follow every second one, and the second of them is agreed with
        step.inp.tokens[a + 1:a + n:2] = 1
        step.parents[a + 1:a + n] = torch.arange(n - 1) // 2 * 2
    step.parents_of = [step.parents[a:a + n].tolist() for a, n in zip(step.cu.tolist(), step.counts)]
    step.inp.kv_lens[2] = 5
    step.inp.block_tables[1, 4] = -3
    step.inp.block_tables[0, 3] = 10 ** 6
    step.inp.block_tables = step.inp.block_tables[:, :5].contiguous()
    caches = [torch.randn(step.blocks, 4, 3), torch.randn(step.blocks - 3, 4, 8)]
    want, moved = [c.clone() for c in caches], 0
    for i, n in enumerate(step.counts):
        a, base = int(step.cu[i]), int(step.inp.kv_lens[i]) - n
        rows = oracle.accepted_path(step.inp.tokens[a:a + n].tolist(), step.parents_of[i], target[a:a + n].tolist(), 19)
        for j, r in enumerate(rows):
            s, d = base + r, base + j
            if min(s, d) >= 0 and max(s, d) < 20:
                (b0, o0), (b1, o1) = step.place(i, s), step.place(i, d)
                for c, w in zip(caches, want):
                    if 0 <= b0 < len(c) and 0 <= b1 < len(c):
                        moved += s != d
                        w[b1, o1] = c[b0, o0]
    assert moved > 5 and step.inp.block_tables.shape[1] == 5
    dev = [c.cuda() for c in caches]
    ops.accept_tree(target.cuda(), step.to("cuda"), step.parents.cuda(), dev)
    assert all(torch.equal(c.cpu(), w) for c, w in zip(dev, want))

@pytest.mark.parametrize("Hq,D", [(16, 64), (12, 128)])
def test_tree_attention_many_pieces_of_one_and_two_row_tiles(Hq, D):
    """A stretch of many short items, with one and with two row tiles in any order, and items of more row tiles than two."""
    counts = [(i * 7) % 23 if i % 29 else 40 for i in range(300)]
    step = oracle.Step([(i * 13) % 150 for i in range(300)], counts, 16, seed=10)
    check_attention(step, Hq, 1, D, torch.bfloat16)
    check_attention(step, Hq, 1, D, torch.bfloat16, window=33)
