"""Bindings of the kernels of a step with trees of drafted tokens (`csrc/cuda/tree_step.cu`, `attention_tree.cu`, `logit_rules.cu`)."""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import cuda_ops
from .reference import TREE_MAX_ROWS, StepRows

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
_SIGNATURES = {
    "xl_step_rows": [_P] * 12 + [_I] * 8 + [_P],
    "xl_accept_tree": [_P] * 9 + [_I] * 5 + [_P] * 3 + [_I] * 2 + [_P],
    "xl_attention_tree": [_P] * 10 + [_I] * 9 + [_L] * 2 + [_F] + [_I] * 4 + [_P, _L, _P],
    "xl_adjust_logits": [_P] + [_I] * 3 + [_L] + [_P] * 2 + [_I] * 3 + [_P, _L, _I] + [_P] * 10 + [_I, _P, _I, _I, _P, _P],
}
_ready = set()


def _launch(device: torch.device, name: str, *args) -> None:
    """Calls an entry point on the current stream of the tensors' own device."""
    L = cuda_ops.lib()
    if name not in _ready:
        getattr(getattr(L, "_real", L), name).argtypes = _SIGNATURES[name]
        _ready.add(name)
    here = device.index is None or device.index == torch.cuda.current_device()
    with contextlib.nullcontext() if here else torch.cuda.device(device):
        cuda_ops._check(getattr(L, name)(*args, torch.cuda.current_stream().cuda_stream), name)
    cuda_ops.launch_count += 1


_sm_counts = {}


def _sms(device: torch.device) -> int:
    n = _sm_counts.get(device)
    if n is None:
        n = _sm_counts[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


def _ptr(t):
    return None if t is None else t.data_ptr()


def step_rows(tables, lens, seqs, counts, n_rows, block_size, parents, max_q, max_blocks) -> StepRows:
    B, words = seqs.numel(), 0 if parents is None else -(-max_q // 64)
    dev = tables.device
    # one allocation for the small outputs
    ints = torch.empty(3 * n_rows + 2 * B + 1, dtype=torch.int32, device=dev)
    positions, slots, token_seq, q_cu, kv_lens = ints.split([n_rows, n_rows, n_rows, B + 1, B])
    out = torch.empty((B, max_blocks), dtype=torch.int32, device=dev)
    tree = None if parents is None else torch.empty((n_rows, words), dtype=torch.int64, device=dev)
    _launch(dev, "xl_step_rows", tables.data_ptr(), lens.data_ptr(), seqs.data_ptr(), counts.data_ptr(), _ptr(parents), positions.data_ptr(),
            slots.data_ptr(), token_seq.data_ptr(), q_cu.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), _ptr(tree), tables.shape[0],
            tables.stride(0), B, n_rows, max_q, max_blocks, block_size, words)
    return StepRows(positions, slots, token_seq, q_cu, kv_lens, out, tree)


def tree_attention(q, k_cache, v_cache, inp, tree, scale, window) -> torch.Tensor:
    T, Hq, D = q.shape
    out = torch.empty((T, Hq * D), dtype=q.dtype, device=q.device)
    block, Hkv = k_cache.shape[1], k_cache.shape[2]
    f32, work, ctas, size = q.dtype == torch.float32, None, 0, 0
    if not f32 and scale > 0:
        # one CTA per SM, fewer where there are fewer key tiles (of 64 keys for up to 128 rows) than it takes to be worth one
        tiles = (inp.max_kv // 64 + 1) * Hkv * (inp.n_seqs + T * (Hq // Hkv) // 128)
        ctas = max(1, min(_sms(q.device), tiles // 4))
        size = cuda_ops.lib().xl_attention_tree_workspace(block, Hq, Hkv, D, inp.max_q, 0, ctas)
    if size:
        if q.stride(2) != 1 or q.stride(1) % 8 or q.stride(0) % max(8, q.stride(1)) or q.data_ptr() % 16:
            q = q.contiguous()
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
    elif q.stride(2) != 1:
        q = q.contiguous()
    bt = inp.block_tables
    _launch(q.device, "xl_attention_tree", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), inp.q_cu.data_ptr(),
            inp.kv_lens.data_ptr(), bt.data_ptr(), inp.token_seq.data_ptr(), inp.positions.data_ptr(), tree.data_ptr(), T, inp.n_seqs, bt.shape[1],
            block, k_cache.shape[0], Hq, Hkv, D, tree.shape[1], q.stride(0), q.stride(1), scale, window, int(f32), inp.max_q, ctas, _ptr(work), size)
    if size:
        cuda_ops.launch_count += 1                               # the join of pieces
    return out


def adjust_logits(logits, q_cu, seqs, history, penalties, tokens, parents, bias, mask, max_q) -> torch.Tensor:
    S, V = logits.shape
    text, lens, prompts = history if history is not None else (None, None, None)
    rep, freq, pres = penalties if history is not None else (None, None, None)
    cu, ids, values = bias if bias is not None else (None, None, None)
    words, mask_of = mask if mask is not None else (None, None)
    B = q_cu.numel() - 1
    pool = lens.numel() if lens is not None else cu.numel() - 1 if cu is not None else B
    _launch(logits.device, "xl_adjust_logits", logits.data_ptr(), int(logits.dtype == torch.float32), S, V, logits.stride(0), q_cu.data_ptr(),
            _ptr(seqs), B, pool, max_q, _ptr(text), 0 if text is None else text.stride(0), 0 if text is None else text.shape[1], _ptr(lens),
            _ptr(prompts), _ptr(rep), _ptr(freq), _ptr(pres), _ptr(tokens if history is not None else None), _ptr(parents), _ptr(cu), _ptr(ids),
            _ptr(values), 0 if ids is None else ids.numel(), _ptr(words), 0 if words is None else words.stride(0),
            0 if words is None else words.shape[0], _ptr(mask_of))
    return logits


def accept_tree(target, inp, parents, caches, depth):
    B, n = inp.n_seqs, len(caches)
    # the widest unit that divides every cache's rows and address
    rows = [c.numel() // max(1, c.shape[0] * c.shape[1]) * c.element_size() for c in caches]
    all_ = 0
    for c, r in zip(caches, rows):
        all_ |= c.data_ptr() | r
    unit = next(u for u in (16, 4, 2, 1) if all_ % u == 0)
    dev = target.device
    out, path = torch.empty((2, B, depth + 1), dtype=torch.int32, device=dev).unbind(0)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    bt = inp.block_tables
    _launch(dev, "xl_accept_tree", target.data_ptr(), inp.tokens.data_ptr(), parents.data_ptr(), inp.q_cu.data_ptr(), inp.kv_lens.data_ptr(),
            bt.data_ptr(), out.data_ptr(), accepted.data_ptr(), path.data_ptr(), target.numel(), B, bt.shape[1], inp.block_size, depth,
            (_P * n)(*[c.data_ptr() for c in caches]), (_I * n)(*[r // unit for r in rows]), (_I * n)(*[c.shape[0] for c in caches]), n, unit)
    return out, accepted, path
