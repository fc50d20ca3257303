"""Operators of a step with trees of drafted tokens on the CPU at the edges of what their documentation allows."""
import os
import sys
import types

import pytest
import torch

import oracle_tree as oracle
from test_tree_step_cpu import acceptance, attention_inputs, rules
from xllm_wxh_b200 import ops
from xllm_wxh_b200.framework.step_input import TreeStep


def test_adjust_logits_refuses_parts_that_are_missing():
    r = rules(40, 3, [2, 1, 1], 4)
    ok = dict(logits=r.logits, q_cu=r.cu, seqs=r.seqs, history=r.history, penalties=r.penalties, tokens=r.tokens, parents=r.parents, bias=r.bias, mask=r.mask)
    kept = r.logits.clone()
    for name in ("history", "penalties", "mask", "bias"):
        for missing in range(len(ok[name])):
            part = tuple(None if j == missing else t for j, t in enumerate(ok[name]))
            with pytest.raises(AssertionError):
                ops.adjust_logits(**{**ok, name: part})
    assert torch.equal(r.logits, kept)


@pytest.mark.parametrize("window", [1, 40, 150])
def test_tree_attention_window_with_positions_of_any_kind(window):
    """A row's position counts as one of its sequence's rows': the nearest one."""
    step = oracle.Step([0, 5, 64, 200], [9, 30, 3, 64], 16, seed=4, deep=True, junk_tables=False)
    q, k, v = attention_inputs(step, 4, 2, 16, torch.float32)
    given = step.inp.positions + torch.randint(-400, 400, (step.T,), generator=torch.Generator().manual_seed(window), dtype=torch.int32)
    given[3], given[50] = 2 ** 31 - 1, -2 ** 31
    counts = torch.tensor(step.counts)
    first = torch.repeat_interleave(torch.tensor(step.before), counts).int()
    step.inp.positions = given
    got = ops.tree_attention(q, k, v, step.inp, step.tree, 0.25, window).view(step.T, 4, 16)
    step.inp.positions = given.clamp(first, first + torch.repeat_interleave(counts, counts).int() - 1)
    want, size = oracle.attention(q, k, v, step, step.tree, 0.25, window)
    assert ((got.double() - want).abs() <= oracle.attention_bound(q, k, want, size, 0.25, 264, torch.float32)).all()


def test_tree_attention_without_table_columns_or_blocks():
    step = oracle.Step([20, 5], [6, 4], 16, seed=3, spare_rows=2, junk_tables=False)
    q, k, v = attention_inputs(step, 4, 2, 8, torch.float32)
    step.inp.block_tables = step.inp.block_tables[:, :0].contiguous()
    assert not ops.tree_attention(q, k, v, step.inp, step.tree, 0.3).any()
    step.inp.kv_lens = torch.zeros_like(step.inp.kv_lens)
    assert not ops.tree_attention(q, k[:0], v[:0], step.inp, step.tree, 0.3).any()


def test_tree_attention_refuses_heads_and_blocks_of_nothing():
    step = oracle.Step([4], [3], 4, junk_tables=False)
    q, k, v = attention_inputs(step, 4, 2, 8, torch.float32)
    for bad in [dict(q=q[:, :0]), dict(q=q[..., :0], k=k[..., :0], v=v[..., :0]), dict(k=k[:, :, :0], v=v[:, :, :0]), dict(k=k[:, :0], v=v[:, :0])]:
        a = {**dict(q=q, k=k, v=v), **bad}
        with pytest.raises(AssertionError):
            ops.tree_attention(a["q"], a["k"], a["v"], step.inp, step.tree, 1.0)


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
    ops.accept_tree(target, step.inp, step.parents, caches)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_chained_drafts_share_one_block_table():
    """Drafts 2 to k of a chain run on the same tables; positions, places and lengths grow by one a draft."""
    from xllm_wxh_b200.runtime.speculative import SpeculativeEngine
    k, bs, ints = 4, 4, lambda *v: torch.tensor(v, dtype=torch.int32)
    tables = torch.arange(1, 3 * 8 + 1, dtype=torch.int32).view(3, 8)
    inp = types.SimpleNamespace(token_seq=ints(1, 1, 0, 2), block_tables=tables, block_size=bs, max_kv=20, layout=types.SimpleNamespace(MB_cap=8))
    seen = []
    draft = types.SimpleNamespace(forward_mtp=lambda mini, kv, h: seen.append(mini) or h + 1)
    engine = types.SimpleNamespace(k=k, draft=draft, draft_kv=None, _propose=lambda h, rows: h[:, 0].int() * 10)
    pos = ints(7, 0, 18)
    out = SpeculativeEngine._chain_drafts(engine, inp, torch.tensor([0, 2, 3]), ints(5, 6, 7), torch.zeros(3, 2), pos)
    assert out.view(3, k).tolist() == [[f, 10, 20, 30] for f in (5, 6, 7)] and pos.tolist() == [7, 0, 18]
    assert len(seen) == k - 1 and len({m.block_tables.data_ptr() for m in seen}) == 1
    for j, m in enumerate(seen):
        at = [p + j for p in (7, 0, 18)]
        assert m.positions.tolist() == at and m.kv_lens.tolist() == [p + 1 for p in at] and m.q_cu.tolist() == [0, 1, 2, 3]
        assert m.slots.tolist() == [int(tables[s, p // bs]) * bs + p % bs for s, p in zip((1, 0, 2), at)]
        assert torch.equal(m.block_tables, tables[[1, 0, 2]]) and m.max_kv == 21 + j


def test_host_extension_is_built_again_for_another_torch_and_other_entry_points(tmp_path, monkeypatch):
    from xllm_wxh_b200 import build_ext
    so, built = tmp_path / "_tree_host.so", []
    monkeypatch.setattr(build_ext, "TREE_HOST_SO", str(so))
    monkeypatch.setattr(build_ext, "_run", lambda cmd, log=None: built.append(cmd))
    build_ext.build_tree_host()
    assert len(built) == 1 and any(torch.__version__ in a for a in built[0])                # missing
    so.write_bytes(b"\0built for torch " + torch.__version__.encode() + b";\0")
    build_ext.build_tree_host()
    assert len(built) == 1                                                                  # as it should be
    api = os.path.join(build_ext.CUDA_DIR, "tree_api.h")
    os.utime(so, (0, os.path.getmtime(api) - 1))
    build_ext.build_tree_host()
    assert len(built) == 2                                                                  # older than the entry points' signatures
    so.write_bytes(b"\0built for torch 1.0;\0")
    build_ext.build_tree_host()
    assert len(built) == 3


def test_host_extension_that_does_not_load_says_why(monkeypatch):
    import xllm_wxh_b200
    from xllm_wxh_b200.ops import cuda_ops, tree_cuda
    monkeypatch.setattr(tree_cuda, "_host", None)
    monkeypatch.setattr(cuda_ops, "lib", lambda: None)
    monkeypatch.delattr(xllm_wxh_b200, "_tree_host", raising=False)
    monkeypatch.setitem(sys.modules, "xllm_wxh_b200._tree_host", None)
    with pytest.raises(RuntimeError, match="does not load .*None in sys.modules.*build_ext"):
        tree_cuda.host()


def test_entry_points_have_one_signature():
    """The host side takes the kernels' argument lists from the header that their definitions include, not from a copy."""
    from xllm_wxh_b200 import build_ext
    from xllm_wxh_b200.ops import tree_cuda
    read = lambda *p: open(os.path.join(*p)).read()
    api = read(build_ext.CUDA_DIR, "tree_api.h")
    for name in tree_cuda._ENTRIES:
        assert f" {name}(" in api and f"decltype(&{name})" in read(build_ext.TREE_HOST_SRC)
    for f in ("tree_step.cu", "attention_tree.cu", "logit_rules.cu"):
        assert '#include "tree_api.h"' in read(build_ext.CUDA_DIR, f)


@pytest.mark.parametrize("shape", [(5,), (7,), (0,), (6, 1)])
def test_tree_step_needs_a_token_for_every_row(shape):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    rows = ops.step_rows(torch.ones(1, 4, dtype=torch.int32), ints(3), ints(0), ints(4), 6, 4, ints(-1, 0, 0, 1, 0, 0), max_q=4)
    with pytest.raises(ValueError):
        TreeStep(torch.zeros(shape, dtype=torch.int32), rows, 4, 4, 7)
    assert TreeStep(torch.zeros(6, dtype=torch.int32), rows, 4, 4, 7).n_tokens == 6
