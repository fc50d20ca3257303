"""Operators of a step with trees of drafted tokens on the CPU at the edges of what their documentation allows."""
import pytest
import torch

from test_tree_step_cpu import rules
from xllm_wxh_b200 import ops


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
