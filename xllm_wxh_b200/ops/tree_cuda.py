"""Kernels of a step with trees of drafted tokens (`csrc/cuda/tree_step.cu`, `attention_tree.cu`, `logit_rules.cu`), called through the
`_tree_host` extension (`csrc/torch/tree_host.cpp`), which looks over the arguments, allocates the outputs and launches on the current
stream of the tensors' device.  Each function returns None when the arguments are not as documented in `ops`."""
from __future__ import annotations

import ctypes

import torch

from . import cuda_ops
from .reference import StepRows

_host = _timed = None
_ENTRIES = ("xl_step_rows", "xl_accept_tree", "xl_attention_tree_workspace", "xl_attention_tree", "xl_adjust_logits")


def host():
    global _host, _timed
    if _host is None:
        L = cuda_ops.lib()
        real = getattr(L, "_real", L)
        try:
            from .. import _tree_host as h
        except ImportError as e:
            raise RuntimeError(f"_tree_host does not load ({e}): run `python -m xllm_wxh_b200.build_ext` (needs g++)") from e
        h.bind({name: ctypes.cast(getattr(real, name), ctypes.c_void_p).value for name in _ENTRIES})
        _host, _timed = h, cuda_ops.kernel_timing()
    return _host


def _call(name, launches, *args):
    f = getattr(_host or host(), name)
    if _timed is not None and _timed.enabled and not torch.cuda.is_current_stream_capturing():
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        out = f(*args)
        e1.record()
        _timed.records.append(("xl_" + name, e0, e1))
    else:
        out = f(*args)
    if out is not None:
        cuda_ops.launch_count += launches
    return out


def step_rows(*args):
    out = _call("step_rows", 1, *args)
    return None if out is None else StepRows._make(out)


def tree_attention(q, k_cache, v_cache, inp, tree, scale, window):
    # with the join of split keys (a step of one key tile needs none)
    return _call("tree_attention", 2, q, k_cache, v_cache, inp.q_cu, inp.kv_lens, inp.block_tables, inp.token_seq, inp.positions, inp.n_seqs, inp.max_q,
                 inp.max_kv, tree, scale, window)


def adjust_logits(logits, q_cu, seqs, history, penalties, tokens, parents, bias, mask, max_q):
    n = (history is not None or bias is not None) + (mask is not None)
    return _call("adjust_logits", n, logits, q_cu, seqs, *history or (None,) * 3, *penalties or (None,) * 3, tokens, parents, *bias or (None,) * 3,
                 *mask or (None,) * 2, max_q)


def accept_tree(target, inp, parents, caches, depth):
    return _call("accept_tree", max(1, -(-len(caches) // 128)), target, inp.tokens, parents, inp.q_cu, inp.kv_lens, inp.block_tables, inp.n_seqs,
                 inp.block_size, inp.max_q, depth, caches)
