"""Kernels of a step with trees of drafted tokens against their definitions in 64 bits (floating outputs) and the CPU forms (whole
numbers): sizes, layouts and masks where they can go wrong, other streams, captured graphs."""
import types

import numpy as np
import pytest
import torch

import oracle_tree as oracle
from test_tree_step_cpu import acceptance, attention_inputs, check_acceptance, check_rules, expected_acceptance, rules
from xllm_wxh_b200 import ops
from xllm_wxh_b200.ops import cuda_ops

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.fixture(autouse=True)
def status():
    yield
    assert cuda_ops.read_status() == 0


def cuda(x):
    return x.cuda() if isinstance(x, torch.Tensor) else tuple(map(cuda, x)) if isinstance(x, (tuple, list)) else x


def captured(f):
    """f's outputs from a graph captured around it (after one plain run), and the graph."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return out, g


# ----------------------------------------------------------------------------- step_rows
@pytest.mark.parametrize("B,counts_to,MB,block,tree,pad", [(1, 1, 1, 1, False, 0), (1, 256, 40, 16, True, 0), (3, 0, 7, 16, True, 1), (37, 65, 300, 8, True, 5),
                                                           (300, 3, 33, 128, False, 40), (5, 5000, 2050, 16, False, 0), (1100, 9, 5, 24, True, 3)])
def test_step_rows(B, counts_to, MB, block, tree, pad):
    rng = np.random.default_rng(B)
    pool = B + 4
    tables = torch.from_numpy(rng.integers(1, 2 ** 20, (pool, MB + 3)).astype(np.int32))[:, :MB]          # rows of a wider table
    counts = torch.from_numpy(rng.integers(0, counts_to + 1, B).astype(np.int32))
    lens = torch.from_numpy(rng.integers(0, max(1, MB * block - counts_to), pool).astype(np.int32))
    seqs = torch.from_numpy(rng.permutation(pool)[:B].astype(np.int32))
    seqs[:pad] = -1
    n_rows = int(counts.sum()) + 5
    parents = torch.from_numpy(rng.integers(-1, max(1, counts_to), n_rows).astype(np.int32)) if tree else None   # some name no earlier row
    for rows in (n_rows, max(0, n_rows - 9)):                                                              # fewer rows than counted: cut off
        args = (tables, lens, seqs, counts, rows, block, parents[:rows] if tree else None, max(1, counts_to))
        want = ops.step_rows(*args)
        got = ops.step_rows(tables.cuda().as_strided(tables.shape, (MB, 1)) if MB == 1 else cuda(tables), *map(cuda, args[1:4]), rows, block, cuda(args[6]),
                            args[7])
        for name, a, b in zip(want._fields, got, want):
            assert (a is None and b is None) or torch.equal(a.cpu(), b), name


def test_step_rows_past_the_table():
    got = ops.step_rows(torch.ones(1, 2, dtype=I32).cuda(), *cuda((torch.tensor([7], dtype=I32), torch.tensor([0], dtype=I32), torch.tensor([4], dtype=I32))), 4, 4)
    assert got.slots.tolist() == [7, 1, 2, 3] and got.block_tables.tolist() == [[1, 1]]                     # places past the table: the reserved block


@pytest.mark.parametrize("cut", [lambda t: t[:, 3:7], lambda t: t[:1, 3:7].expand(3, 4)])
def test_step_rows_columns_of_a_wider_table(cut):
    """Places past the columns that were given are past the table, whatever lies behind them in memory."""
    base = torch.arange(1, 25, dtype=I32).view(3, 8)
    rest = torch.tensor([14, 3, 9], dtype=I32), torch.tensor([2, 0, 1], dtype=I32), torch.tensor([9, 4, 8], dtype=I32)
    want = ops.step_rows(cut(base), *rest, 24, 4)
    got = ops.step_rows(cut(base.cuda()), *cuda(rest), 24, 4)
    for a, b in zip(got[:6], want[:6]):
        assert torch.equal(a.cpu(), b)


# ----------------------------------------------------------------------------- attention
def check_attention(step, Hq, Hkv, D, dtype, window=-1, tree=None, seed=0, scale=None, change=None, layout="dense"):
    scale = D ** -0.5 if scale is None else scale
    q, k, v = attention_inputs(step, Hq, Hkv, D, dtype, seed)
    tree = step.tree if tree is None else tree
    if change is not None:
        change(q, k, v)
    held = [torch.zeros(0)]
    if layout == "rows":                                         # a view of a projection's wider rows
        wide = torch.randn(step.T, (Hq + 2 * Hkv) * D).to(dtype)
        wide[:, :Hq * D] = q.flatten(1)
        held = [wide.cuda()]
        dq = held[0][:, :Hq * D].view(step.T, Hq, D)
    elif layout == "heads":                                      # head-major
        dq = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    elif layout == "odd":                                        # rows on no 16-byte boundary
        held = [torch.zeros(step.T, Hq * D + 1, dtype=dtype).cuda()]
        dq = held[0][:, 1:].view(step.T, Hq, D) if step.T == 1 else held[0].as_strided((step.T, Hq, D), (Hq * D + 1, D, 1), 1)
        dq.copy_(q)
    elif layout == "columns":                                    # columns apart
        dq = q.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    else:
        dq = q.cuda()
    got = ops.tree_attention(dq, k.cuda(), v.cuda(), step.to("cuda"), tree.cuda(), scale, window).view(step.T, Hq, D).cpu().double()
    want, size = oracle.attention(q, k, v, step, tree, scale, window)
    longest = max(b + n for b, n in zip(step.before, step.counts)) if step.before else 0
    bound = oracle.attention_bound(q, k, want, size, scale, longest, dtype)
    nan = want.isnan()
    assert torch.equal(nan, got.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    fine = ~nan & ~inf
    off = ((got - want).abs() - bound)[fine]
    assert not off.numel() or off.max() <= 0, (float(off.max()), float((got - want).abs()[fine].max()))
    return got


SIZES = [                     # before, counts, Hq, Hkv, D, block, words
    ([0], [1], 8, 2, 128, 16, 1),
    ([1], [1], 4, 4, 64, 128, 1),
    ([63, 64, 65], [1, 2, 3], 8, 2, 128, 64, 1),
    ([0, 300, 7], [64, 17, 5], 32, 8, 128, 16, 1),
    ([1000, 0, 129, 2], [9, 4, 0, 33], 28, 4, 64, 16, 1),
    ([500], [65], 16, 2, 128, 128, 2),
    ([70, 3], [256, 130], 8, 4, 64, 32, 4),
    ([2500], [16], 8, 1, 128, 128, 1),
    ([200, 30], [12, 7], 40, 8, 128, 16, 1),
    ([200, 30], [12, 7], 48, 1, 128, 16, 1),
    ([200, 30], [3, 7], 160, 1, 64, 16, 1),
    ([90, 40], [12, 7], 6, 2, 80, 8, 1),
    ([90, 40], [12, 7], 6, 2, 40, 24, 1),
    ([90, 40], [12, 7], 6, 6, 8, 48, 1),
    ([90, 40], [12, 7], 6, 2, 192, 16, 1),
    ([90, 40], [12, 7], 6, 2, 256, 16, 1),
    ([90, 40], [12, 7], 4, 2, 512, 16, 1),
    ([90, 40], [12, 7], 6, 2, 7, 5, 1),
    ([90, 40], [12, 7], 6, 2, 64, 1, 1),
    ([300], [1], 1, 1, 64, 16, 1),                               # an odd number of partial rows
    ([700], [3], 3, 1, 68, 16, 1),
    (list(range(0, 400, 10)), [1 + i % 6 for i in range(40)], 8, 2, 64, 16, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("before,counts,Hq,Hkv,D,block,words", SIZES)
def test_tree_attention(before, counts, Hq, Hkv, D, block, words, dtype):
    step = oracle.Step(before, counts, block, seed=len(before), words=words, spare_rows=3)
    check_attention(step, Hq, Hkv, D, dtype)


@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 333])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (64, torch.float32)])
def test_tree_attention_window(window, D, dtype):
    step = oracle.Step([0, 5, 64, 200, 700], [9, 30, 3, 64, 12], 16, seed=4, deep=True)
    check_attention(step, 8, 2, D, dtype, window)


@pytest.mark.parametrize("layout", ["rows", "heads", "odd", "columns"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_layouts_of_q(layout, dtype):
    check_attention(oracle.Step([130, 20], [6, 11], 16, seed=5, spare_rows=1), 8, 2, 64, dtype, layout=layout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_masks_of_any_kind(dtype):
    step = oracle.Step([0, 70, 129], [5, 64, 70], 16, seed=6, words=2)
    tree = torch.randint(-2 ** 62, 2 ** 62, step.tree.shape, generator=torch.Generator().manual_seed(0))
    tree[1], tree[7] = 0, 0                                      # nothing at all; cached tokens only
    got = check_attention(step, 8, 2, 128, dtype, tree=tree)
    assert not got[1].any()
    check_attention(step, 8, 2, 128, dtype, tree=tree, window=40)
    tree.zero_()
    check_attention(oracle.Step([0], [9], 16, seed=6), 8, 2, 64, dtype, tree=tree[:9, :1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_tree_attention_bad_values_behind_masks(bad, dtype):
    """Whatever stands in masked places (rows of other branches, places behind the last row, keys ahead of the window) changes nothing."""
    value = torch.finfo(dtype).min if bad == "lowest" else bad
    for before, n, window in [(70, 10, -1), (3, 70, -1), (300, 12, 50), (128, 4, -1), (60, 3, -1)]:
        step = oracle.Step([before, 9], [n, 2], 16, seed=7, words=2)

        def change(q, k, v):
            used = torch.zeros(step.blocks, step.block, dtype=torch.bool)
            for i, (b, m) in enumerate(zip(step.before, step.counts)):
                for p in range(b + m):
                    used[step.place(i, p)] = True
            k[~used], v[~used] = value, value
            if window > 0:
                for p in range(before - window - 2):
                    k[step.place(0, p)], v[step.place(0, p)] = value, value
        check_attention(step, 8, 2, 128, dtype, window=window, change=change)
        # one row of the tree is bad: only the rows that see it notice
        if bad != "lowest":
            def worse(q, k, v):
                change(q, k, v)
                v[step.place(0, before + n - 1)][..., 3] = value
                v[step.place(0, before + 1)][..., 5] = value
            check_attention(step, 8, 2, 128, dtype, window=window, change=worse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_large_and_small_scores(dtype):
    step = oracle.Step([400, 3], [20, 30], 16, seed=8)

    def peaked(q, k, v):
        q.mul_(20)
    check_attention(step, 8, 2, 64, dtype, change=peaked)

    def growing(q, k, v):                                        # the running maximum grows by much, again and again
        q.fill_(1)
        for p in range(400):
            k[step.place(0, p)] = p / 40
    check_attention(step, 8, 2, 64, dtype, change=growing)

    def far_below(q, k, v):
        q.fill_(1)
        k.fill_(-200)
    check_attention(step, 8, 2, 64, dtype, change=far_below)
    check_attention(step, 8, 2, 64, dtype, scale=0.0)


@pytest.mark.parametrize("before,counts,Hq,Hkv,D", [([9000], [5], 8, 2, 128), ([5000, 20, 3000], [64, 64, 1], 32, 4, 64), ([4000], [3], 2, 2, 128)])
def test_tree_attention_long_contexts(before, counts, Hq, Hkv, D):
    step = oracle.Step(before, counts, 128, seed=9)
    a = check_attention(step, Hq, Hkv, D, torch.bfloat16)
    assert torch.equal(a, check_attention(step, Hq, Hkv, D, torch.bfloat16))          # bit for bit


def test_tree_attention_many_short_sequences():
    step = oracle.Step([i % 50 for i in range(700)], [i % 3 for i in range(700)], 16, seed=10)
    check_attention(step, 4, 2, 64, torch.bfloat16)


def test_tree_attention_empty_steps():
    for before, counts in [([], []), ([5, 6], [0, 0])]:
        step = oracle.Step(before, counts, 16, spare_rows=2)
        q, k, v = attention_inputs(step, 4, 2, 64, torch.bfloat16)
        assert not ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), 1.0).any()
    step = oracle.Step([5], [0], 16)
    q, k, v = attention_inputs(step, 4, 2, 64, torch.bfloat16)
    assert ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), 1.0).shape == (0, 256)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_attention_rows_ahead_of_the_first_sequence_and_without_keys(dtype):
    """Rows that no sequence owns lie ahead of the first one too; a sequence without keys gets zeros."""
    step = oracle.Step([20, 5], [6, 4], 16, seed=3)
    q, k, v = attention_inputs(step, 4, 2, 64, dtype)
    inp = step.to("cuda")
    inp.q_cu = inp.q_cu + 3
    pad = lambda t: torch.cat([t[:1].expand(3, *t.shape[1:]), t])
    inp.token_seq, inp.positions = pad(inp.token_seq), pad(inp.positions)
    inp.kv_lens = inp.kv_lens * torch.tensor([1, 0], dtype=I32).cuda()
    got = ops.tree_attention(pad(q).cuda(), k.cuda(), v.cuda(), inp, pad(step.tree).cuda(), 0.3).view(13, 4, 64).cpu().double()
    want, size = oracle.attention(q, k, v, step, step.tree, 0.3)
    assert not got[:3].any() and not got[9:].any()
    assert ((got[3:9] - want[:6]).abs() <= oracle.attention_bound(q, k, want, size, 0.3, 26, dtype)[:6]).all()


def test_tree_attention_places_past_32_bits():
    """A cache of more than 2^32 elements: keys and values at its far end."""
    block, Hkv, D = 128, 16, 128
    blocks = 2 ** 32 // (block * Hkv * D) + 40
    k = torch.zeros(blocks, block, Hkv, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    small = oracle.Step([300], [6], block, seed=11, junk_tables=False)
    q, ks, vs = attention_inputs(small, 16, Hkv, D, torch.bfloat16)
    k[-small.blocks:], v[-small.blocks:] = ks.cuda(), vs.cuda()
    inp = small.to("cuda")
    inp.block_tables = inp.block_tables + (blocks - small.blocks)
    got = ops.tree_attention(q.cuda(), k, v, inp, small.tree.cuda(), 0.1).view(6, 16, D).cpu().double()
    want, size = oracle.attention(q, ks, vs, small, small.tree, 0.1)
    assert ((got - want).abs() <= oracle.attention_bound(q, ks, want, size, 0.1, 306, torch.bfloat16)).all()


def test_tree_attention_replayed_with_other_lengths_and_on_another_stream():
    """Two graphs of the same sizes, replayed in turn and at once on two streams with lengths that change in between; the launches go by the bounds."""
    for D, dtype in [(128, torch.bfloat16), (64, torch.float32)]:
        a, b = oracle.Step([40, 900], [7, 9], 16, seed=12), oracle.Step([900, 35], [9, 7], 16, seed=13)
        sides = []
        for step in (a, b):
            q, k, v = attention_inputs(step, 8, 2, D, dtype, seed=step.before[0])
            inp = step.to("cuda")
            inp.max_kv, inp.max_q = 1000, 16
            dq, dk, dv, tree = q.cuda(), k.cuda(), v.cuda(), step.tree.cuda()
            out, g = captured(lambda: ops.tree_attention(dq, dk, dv, inp, tree, 0.2))
            want, size = oracle.attention(q, k, v, step, step.tree, 0.2)
            sides.append((out, g, want, oracle.attention_bound(q, k, want, size, 0.2, 909, dtype), inp, tree, dq, dk, dv))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(3):
            for s, side in zip(streams, sides):
                with torch.cuda.stream(s):
                    side[1].replay()
        torch.cuda.synchronize()
        for out, _, want, bound, *_ in sides:
            assert ((out.view(want.shape).cpu().double() - want).abs() <= bound).all()
        # the first graph's tensors take a step with other lengths
        step = oracle.Step([100, 3], [10, 6], 16, seed=14)
        q, k, v = attention_inputs(step, 8, 2, D, dtype, seed=3)
        out, g, _, _, inp, tree, dq, dk, dv = sides[0]
        dq.copy_(q)
        dk[:step.blocks], dv[:step.blocks] = k.cuda(), v.cuda()
        tree.copy_(step.tree)
        for name in ("q_cu", "kv_lens", "token_seq", "positions"):
            getattr(inp, name).copy_(getattr(step.inp, name))
        inp.block_tables[:, :step.inp.block_tables.shape[1]].copy_(step.inp.block_tables)
        g.replay()
        want, size = oracle.attention(q, k, v, step, step.tree, 0.2)
        assert ((out.view(want.shape).cpu().double() - want).abs() <= oracle.attention_bound(q, k, want, size, 0.2, 200, dtype)).all()


def test_tree_attention_of_a_chain_is_paged_attention():
    """Rows that follow one another are what `paged_attention` serves."""
    step = oracle.Step([200, 31], [6, 9], 16, seed=15)
    for i, n in enumerate(step.counts):
        step.parents_of[i] = list(range(-1, n - 1))
        a = int(step.cu[i])
        step.tree[a:a + n] = oracle.bits(step.parents_of[i], 1)
    q, k, v = attention_inputs(step, 8, 2, 128, torch.bfloat16)
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), step.to("cuda"), step.tree.cuda(), 0.1)
    from xllm_wxh_b200.ops import reference as ref
    want = ref.paged_attention(q, k, v, step.inp.q_cu, step.inp.kv_lens, step.inp.block_tables.clamp(max=step.blocks - 1), 2, 0.1)
    w, size = oracle.attention(q, k, v, step, step.tree, 0.1)
    bound = oracle.attention_bound(q, k, w, size, 0.1, 206, torch.bfloat16).flatten(1)
    assert ((got.cpu().double() - want.double()).abs() <= 2 * bound).all()


# ----------------------------------------------------------------------------- logits
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,rows_of,masked,tree", [(1, [1], True, False), (50, [1, 1, 1], True, False), (97, [4, 0, 9], True, True), (64, [3], False, True),
                                                   (33, [64, 2], True, True), (1000, [200, 1, 30], True, True), (40000, [2, 1], True, True)])
def test_adjust_logits(V, rows_of, masked, tree, dtype):
    if V == 40000:                                               # the mask of one column at a time is slow to state
        masked = False
    r = rules(V, len(rows_of) + 2, rows_of, V, dtype, masked, tree)
    most = max(rows_of)
    for pad in (0, 3):                                           # rows of a wider tensor: no alignment
        wide = torch.randn(len(r.logits), V + pad).to(dtype)
        wide[:, :V] = r.logits
        wide_d = wide.cuda()
        got = wide_d[:, :V]
        assert ops.adjust_logits(got, *cuda((r.cu, r.seqs, r.history, r.penalties, r.tokens, r.parents, r.bias, r.mask)), max_q=most) is got
        check_rules(r, got.cpu(), dtype)
        assert torch.equal(wide_d[:, V:].cpu(), wide[:, V:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adjust_logits_parts(dtype):
    """Each part alone, and nothing at all."""
    r = rules(500, 6, [3, 5, 2], 3, dtype)
    none = dict(history=None, penalties=None, tokens=None, parents=None, bias=None, mask=None)
    for parts in [(), ("history", "penalties"), ("history", "penalties", "tokens"), ("history", "penalties", "tokens", "parents"), ("bias",), ("mask",),
                  ("bias", "mask")]:
        some = types.SimpleNamespace(**{**vars(r), **none, **{p: getattr(r, p) for p in parts}})
        got = r.logits.cuda()
        ops.adjust_logits(got, *cuda((some.cu, some.seqs, some.history, some.penalties, some.tokens, some.parents, some.bias, some.mask)))
        if "history" in parts or "bias" in parts:
            check_rules(some, got.cpu(), dtype)
        elif "mask" in parts:
            some.bias = (torch.zeros(7, dtype=I32), torch.zeros(0, dtype=I32), torch.zeros(0))
            check_rules(some, got.cpu(), dtype)
        else:
            assert torch.equal(got.cpu(), r.logits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,length,distinct,biases", [(40000, 5000, 4990, 10), (40000, 20000, 15000, 300), (40000, 7, 3, 30000), (300, 100000, 300, 0), (9000, 8192, 8192, 0)])
def test_adjust_logits_long_histories(V, length, distinct, biases, dtype):
    """More ids than the table holds at a time, long lists of biases, one id a hundred thousand times."""
    g = torch.Generator().manual_seed(length)
    distinct = min(distinct, V)
    ids = torch.randint(0, distinct, (2, length), generator=g, dtype=I32) * (V // distinct)
    ids[0] = 7 % V
    lens, prompts = torch.tensor([length, length], dtype=I32), torch.tensor([length // 3, 0], dtype=I32)
    pen = (torch.tensor([1.3, 0.7]), torch.tensor([0.01, -0.02]), torch.tensor([0.5, 0.1]))
    tokens, parents = torch.randint(0, V, (6,), generator=g, dtype=I32), torch.tensor([-1, 0, 0, -1, 0, 1], dtype=I32)
    tokens[1], tokens[4] = 7 % V, int(ids[1, 5])
    bias = (torch.tensor([0, 0, biases], dtype=I32), torch.randint(0, V, (biases,), generator=g, dtype=I32), torch.randn(biases, generator=g)) if biases else None
    x = (torch.randn(6, V, generator=g) * 3).to(dtype)
    got = x.cuda()
    cu = torch.tensor([0, 3, 6], dtype=I32)
    ops.adjust_logits(got, *cuda((cu, None, (ids, lens, prompts), pen, tokens, parents, bias)), max_q=3)
    y = x.double()
    for b in range(2):
        seen, made = torch.bincount(ids[b].long(), minlength=V), torch.bincount(ids[b, int(prompts[b]):].long(), minlength=V)
        add = torch.zeros(V, dtype=torch.float64)
        if bias is not None and b == 1:
            for i, v in zip(bias[1].tolist(), bias[2].tolist()):
                add[i] = v
        rep, freq, pres = (float(t[b].double()) for t in pen)
        for r in range(3 * b, 3 * b + 3):
            mine = torch.bincount(tokens[[3 * b + j for j in oracle.line(parents[3 * b:3 * b + 3].tolist(), r - 3 * b)]].long(), minlength=V)
            n = (made + mine).double()
            z = y[r] - n * freq - (n > 0) * pres
            y[r] = torch.where(seen + mine > 0, torch.where(z < 0, z * rep, z / rep), y[r]) + add
            # five roundings of fp32 to values of at most this size
            big = (x[r].double().abs() + n * abs(freq) + abs(pres)) * max(rep, 1 / rep) + add.abs()
            bound = 2.0 ** -24 * 6 * big + (y[r].abs() * 2.0 ** -8 * 1.01 if dtype == torch.bfloat16 else 0)
            assert ((got[r].cpu().double() - y[r]).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adjust_logits_masks_of_a_large_vocabulary(dtype):
    V, S, g = 50257, 5, torch.Generator().manual_seed(1)
    x = torch.randn(S, V, generator=g).to(dtype)
    x[1, 10], x[2, 20], x[3, 30] = float("nan"), float("inf"), -float("inf")
    words = torch.randint(-2 ** 31, 2 ** 31, (4, -(-V // 32) + 1), generator=g, dtype=torch.int64).int()
    words[1], words[2, ::3], words[2, 1::3] = 0, 0, -1
    of = torch.tensor([2, 1, 0, -1, 9], dtype=I32)                                    # 9: no such mask, none
    got = x.cuda()
    ops.adjust_logits(got, torch.arange(S + 1, dtype=I32).cuda(), mask=(words.cuda()[:, :-1], of.cuda()))
    allowed = ((words[..., None] >> torch.arange(32).int()) & 1).flatten(1)[:, :V].bool()
    for r in range(S):
        want = x[r].masked_fill(~allowed[of[r]], -float("inf")) if of[r] in (0, 1, 2) else x[r]
        assert torch.equal(got[r].cpu().nan_to_num(5.0), want.nan_to_num(5.0)) and torch.equal(got[r].cpu().isnan(), want.isnan())


def test_adjust_logits_special_values():
    """Infinities and NaN go through the formula; the same inputs give the same bits; ids outside the vocabulary are passed over."""
    V = 64
    x = torch.tensor([[float("inf"), -float("inf"), float("nan"), torch.finfo(torch.float32).min, 1.0] + [0.5] * (V - 5)])
    history = (torch.tensor([[0, 1, 2, 3, -5, V, 2 ** 31 - 1, 4, 4]], dtype=I32), torch.tensor([9], dtype=I32), torch.tensor([2], dtype=I32))
    pen = (torch.tensor([2.0]), torch.tensor([0.5]), torch.tensor([0.25]))
    bias = (torch.tensor([0, 4], dtype=I32), torch.tensor([4, -1, V, 4], dtype=I32), torch.tensor([100.0, 1.0, 1.0, -float("inf")]))
    got = x.cuda()
    ops.adjust_logits(got, *cuda((torch.tensor([0, 1], dtype=I32), None, history, pen, None, None, bias)))
    got = got.cpu()[0]
    assert got[0] == float("inf") and got[1] == -float("inf") and got[2].isnan() and got[3] == -float("inf") and got[4] == -float("inf")
    assert torch.equal(got[5:], x[0, 5:])


def test_adjust_logits_replayed():
    r = rules(3000, 9, [4, 1, 7], 8)
    args = cuda((r.cu, r.seqs, r.history, r.penalties, r.tokens, r.parents, r.bias, r.mask))
    x, fresh = r.logits.cuda(), r.logits.cuda()

    def run():
        x.copy_(fresh)
        return ops.adjust_logits(x, *args, max_q=8)
    _, g = captured(run)
    g.replay()
    check_rules(r, x.cpu(), torch.float32)
    args[2][1].sub_(1).clamp_(min=0)                              # other lengths
    r.history[1].sub_(1).clamp_(min=0)
    g.replay()
    check_rules(r, x.cpu(), torch.float32)


# ----------------------------------------------------------------------------- accept_tree
@pytest.mark.parametrize("before,counts,block,depth,vocab", [([0], [1], 4, 0, 3), ([5, 0, 30], [9, 0, 40], 4, 12, 3), ([7, 7], [12, 64], 16, 63, 2), ([2], [30], 8, 2, 2),
                                                             ([100], [256], 128, 255, 1), ([3] * 70, [17] * 70, 1, 16, 2)])
def test_accept_tree(before, counts, block, depth, vocab):
    for seed, deep in [(1, True), (2, False)]:
        step = oracle.Step(before, counts, block, seed=seed, deep=deep, words=4, spare_rows=2)
        target = acceptance(step, seed, vocab)
        g = torch.Generator().manual_seed(seed)
        for shapes in [[(3, 4), (5,)], [(8, 128)] * 3, [(1,)], [(2, 24), (700,)], []]:
            caches = [torch.randn(step.blocks, block, *s, generator=g).to(torch.bfloat16) for s in shapes] + [torch.randint(0, 100, (step.blocks, block, 7), generator=g)]
            if len(shapes) == 1:
                caches = [torch.randint(0, 256, (step.blocks, block, 3), generator=g, dtype=torch.uint8)]
            rows_of, want = expected_acceptance(step, target, caches, depth)
            inp = step.to("cuda")
            dev = [c.cuda() for c in caches]
            check_acceptance(step, target, ops.accept_tree(target.cuda(), inp, step.parents.cuda(), dev, depth), depth, rows_of)
            assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))


def test_accept_tree_many_caches_and_replay():
    step = oracle.Step([4, 50], [20, 11], 8, seed=3, deep=True)
    target = acceptance(step, 5, 2)
    caches = [torch.randn(step.blocks, 8, 16) for _ in range(300)]
    rows_of, want = expected_acceptance(step, target, caches, 19)
    dev, inp, up, t = [c.cuda() for c in caches], step.to("cuda"), step.parents.cuda(), target.cuda()
    keep = [d.clone() for d in dev]

    def run():
        for d, k in zip(dev, keep):
            d.copy_(k)
        return ops.accept_tree(t, inp, up, dev)
    result, g = captured(run)
    g.replay()
    check_acceptance(step, target, result, 19, rows_of)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))


# ----------------------------------------------------------------------------- together
def test_model_goes_on_as_without_drafts():
    from helpers.tree_generation import check_generation
    check_generation("cuda", torch.bfloat16)


def test_a_whole_step_replayed():
    """Maps, attention, rules and acceptance of one step in a graph, replayed for three steps of growing sequences."""
    B, MB, block, Hq, Hkv, D, V, n, pool = 4, 20, 16, 8, 2, 128, 500, 9, 6
    g = torch.Generator().manual_seed(0)
    rng = np.random.default_rng(0)
    tables = (torch.randperm(pool * MB, generator=g).int() + 1).view(pool, MB)
    lens = torch.tensor([40, 0, 7, 130, 255, 16], dtype=I32)
    seqs, counts = torch.tensor([3, 0, -1, 5], dtype=I32), torch.tensor([9, 4, 6, 1], dtype=I32)
    history, prompts = torch.randint(0, V, (pool, 400), generator=g, dtype=I32), torch.tensor([10, 0, 0, 20, 5, 16], dtype=I32)
    pen = tuple(torch.rand(pool, generator=g) + 0.5 for _ in range(3))
    words, of = torch.randint(-2 ** 31, 2 ** 31, (3, 16), generator=g, dtype=torch.int64).int(), torch.randint(-1, 3, (24,), generator=g, dtype=I32)
    parents = torch.tensor(oracle.random_parents(rng, 9) + oracle.random_parents(rng, 4) + [-1] + [0] * 10, dtype=I32)
    tokens = torch.randint(0, 3, (24,), generator=g, dtype=I32)
    q = torch.randn(24, Hq, D, generator=g).bfloat16()
    kc, vc = (torch.randn(pool * MB + 1, block, Hkv, D, generator=g).bfloat16() for _ in range(2))
    x = torch.randn(24, V, generator=g)
    from xllm_wxh_b200.framework.step_input import TreeStep

    def one(tables, lens, seqs, counts, history, prompts, pen, words, of, parents, tokens, q, kc, vc, x):
        rows = ops.step_rows(tables, lens, seqs, counts, 24, block, parents, max_q=n)
        inp = TreeStep(tokens, rows, block, n, MB * block)
        o = ops.paged_attention(q, kc, vc, inp, D ** -0.5)
        y = ops.adjust_logits(x.clone(), inp.q_cu, seqs, (history, lens, prompts), pen, tokens, parents, None, (words, of), n)
        target = y.argmax(-1).int() % 3
        out, accepted, path = ops.accept_tree(target, inp, parents, (kc, vc))
        live = seqs >= 0
        lens.index_add_(0, seqs.clamp(min=0).long(), torch.where(live, accepted + 1, torch.zeros_like(accepted)))
        return *rows, o, y, out, accepted, path
    host = [tables, lens, seqs, counts, history, prompts, pen, words, of, parents, tokens, q, kc, vc, x]
    dev = list(cuda(host))
    saved = [t.clone() for t in (dev[1], dev[12], dev[13])]
    result, graph = captured(lambda: one(*dev))
    for t, s in zip((dev[1], dev[12], dev[13]), saved):
        t.copy_(s)
    for _ in range(3):
        want = one(*host)
        graph.replay()
        for i, (a, b) in enumerate(zip(result, want)):
            if b.is_floating_point():
                a, b = a.cpu().float().nan_to_num(0, 0, 0), b.float().nan_to_num(0, 0, 0)
                assert (a - b).norm() <= 2.0 ** -6 * b.norm(), i                       # two roundings to bf16 on either side
            else:
                assert torch.equal(a.cpu(), b), i
        assert torch.equal(dev[1].cpu(), lens) and torch.equal(dev[12].cpu(), kc) and torch.equal(dev[13].cpu(), vc)


# ----------------------------------------------------------------------------- refusals
def refused(op, ok, bads):
    op(**ok)
    for bad in bads:
        with pytest.raises(AssertionError):
            op(**{**ok, **bad})


def test_refusals():
    i = lambda *v: torch.tensor(v, dtype=I32).cuda()
    tables = torch.ones(2, 4, dtype=I32).cuda()
    refused(ops.step_rows, dict(tables=tables, lens=i(1, 2), seqs=i(0, 1), counts=i(1, 1), n_rows=2, block_size=4, parents=i(-1, -1)),
            [dict(tables=tables.long()), dict(tables=tables.t()), dict(lens=i(1)), dict(lens=i(1, 2).cpu()), dict(seqs=i(0)), dict(counts=i(1, 1).long()),
             dict(n_rows=-1), dict(block_size=0), dict(max_q=0), dict(max_blocks=5), dict(parents=i(0)), dict(max_q=257)])
    step = oracle.Step([4], [3], 16)
    target = acceptance(step, 1).cuda()
    q, k, v = (t.cuda() for t in attention_inputs(step, 4, 2, 64, torch.bfloat16))
    inp, tree = step.to("cuda"), step.tree.cuda()
    other = lambda **kw: types.SimpleNamespace(**{**vars(inp), **kw})
    refused(ops.tree_attention, dict(q=q, k_cache=k, v_cache=v, inp=inp, tree=tree, scale=1.0),
            [dict(q=q.half(), k_cache=k.half(), v_cache=v.half()), dict(q=q.float()), dict(v_cache=v[..., :32].contiguous()), dict(q=q[:, :3]),
             dict(k_cache=k.transpose(1, 2)), dict(k_cache=k.cpu()), dict(tree=tree.int()), dict(tree=tree[:2]),
             dict(tree=torch.zeros(3, 5, dtype=torch.int64).cuda()), dict(inp=other(q_cu=inp.q_cu.long())), dict(inp=other(kv_lens=i(1, 2))),
             dict(inp=other(positions=i(1))), dict(inp=other(max_q=300))])
    x, cu, f = torch.zeros(3, 40).cuda(), i(0, 3), torch.ones(1).cuda()
    history, words = (i(1, 2).view(1, 2), i(2), i(1)), torch.ones(1, 2, dtype=I32).cuda()
    refused(ops.adjust_logits, dict(logits=x, q_cu=cu, history=history, penalties=(f, f, f), tokens=i(1, 2, 3), mask=(words, i(0, 0, 0)),
                                    bias=(i(0, 1), i(4), f)),
            [dict(logits=x.half()), dict(logits=x.t()), dict(q_cu=cu.long()), dict(history=None), dict(penalties=None), dict(penalties=(f, f, f.cpu())),
             dict(tokens=i(1)), dict(tokens=None, parents=i(0, 0, 0)), dict(mask=(words[:, :1], i(0, 0, 0))), dict(mask=(words, i(0))),
             dict(bias=(i(0, 1, 1), i(4), f)), dict(bias=(i(0, 1), i(4), f.double())), dict(seqs=i(0, 0)), dict(max_q=257), dict(max_q=0)])
    n = step.blocks
    caches = torch.zeros(2 * n, 16, 2).cuda()
    parents = step.parents.cuda()
    refused(ops.accept_tree, dict(target=target, inp=inp, parents=parents, caches=[caches[:n], caches[n:]]),
            [dict(target=target.long()), dict(parents=parents[:2]), dict(caches=[caches[:n], caches[n - 1:]]), dict(caches=[caches, caches]),
             dict(caches=[caches.transpose(0, 1)]), dict(caches=[caches.cpu()]), dict(caches=[torch.zeros(2, 8, 2).cuda()]), dict(max_depth=-1),
             dict(max_depth=256), dict(inp=other(max_q=300))])
    torch.cuda.synchronize()


def test_allowed_views():
    """One mask that stands for several by expansion."""
    V = 100
    x = torch.randn(4, V)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, 4), dtype=I32)
    of = torch.tensor([0, 2, -1, 1], dtype=I32)
    want = ops.adjust_logits(x.clone(), torch.tensor([0, 4], dtype=I32), mask=(words.expand(3, 4), of))
    got = ops.adjust_logits(x.cuda(), torch.tensor([0, 4], dtype=I32).cuda(), mask=(words.cuda().expand(3, 4), of.cuda()))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_rows_than_keys(dtype):
    """A step whose lengths name fewer keys than rows: the rows' first keys are the tree's, as on the CPU."""
    step = oracle.Step([0], [5], 16, seed=1)
    q, k, v = attention_inputs(step, 2, 2, 64, dtype)
    inp = types.SimpleNamespace(**{**vars(step.inp), "kv_lens": torch.tensor([3], dtype=I32)})
    want = ops.tree_attention(q, k, v, inp, step.tree, 0.2)
    there = types.SimpleNamespace(**{**vars(step.to("cuda")), "kv_lens": torch.tensor([3], dtype=I32).cuda()})
    got = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), there, step.tree.cuda(), 0.2)
    # fp32: scores of 64 products below 20 in sum of sizes 2^9 are off by 2^-24 x 2^9 x 8 at most, which the weights take over: 2^-12 of
    # values below 8.  bf16: the weights' and the result's roundings besides, 2^-8 each and once more for the CPU's
    bound = 2 ** -9 if dtype is torch.float32 else 2 ** -9 + 3 * 2 ** -8 * 8
    assert ((got.cpu() - want).abs().float() <= bound).all()
