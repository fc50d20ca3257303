"""Bindings of the kernels of a step with trees of drafted tokens (`csrc/cuda/tree_step.cu`, `attention_tree.cu`, `logit_rules.cu`)."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import cuda_ops
from .reference import TREE_MAX_ROWS, StepRows

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
_SIGNATURES = {
    "xl_step_rows": [_P] * 12 + [_I] * 8 + [_P],
    "xl_accept_tree": [_P] * 9 + [_I] * 5 + [_P] * 3 + [_I] * 2 + [_P],
    "xl_attention_tree": [_P] * 10 + [_I] * 9 + [_L] * 2 + [_F] + [_I] * 7 + [_P, _L, _P],
    "xl_adjust_logits": [_P] + [_I] * 3 + [_L] + [_P] * 2 + [_I] * 3 + [_P, _L, _I] + [_P] * 10 + [_I, _P, _I, _I, _P, _P],
}
_entry = {}


def _launch(device: int, name: str, *args) -> None:
    """Calls an entry point on the current stream of the tensors' own device."""
    f = _entry.get(name)
    if f is None or cuda_ops.kernel_timing() is not None:
        L = cuda_ops.lib()
        getattr(getattr(L, "_real", L), name).argtypes = _SIGNATURES[name]
        f = _entry[name] = getattr(L, name)
    if device == torch.cuda.current_device():
        rc = f(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = f(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        cuda_ops._check(rc, name)
    cuda_ops.launch_count += 1


_sm_counts = {}


def _sms(device: int) -> int:
    n = _sm_counts.get(device)
    if n is None:
        n = _sm_counts[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


@functools.lru_cache(maxsize=1024)
def _workspace(*sizes):
    """(bytes, whether the tensor-core kernel serves these sizes)."""
    f, tc = cuda_ops.lib().xl_attention_tree_workspace, _I(0)
    f.restype = _L
    return f(*sizes, ctypes.byref(tc)), bool(tc.value)


def _ptr(t):
    return None if t is None else t.data_ptr()


def step_rows(tables, lens, seqs, counts, n_rows, block_size, parents, max_q, max_blocks) -> StepRows:
    B, words = seqs.numel(), 0 if parents is None else -(-max_q // 64)
    # one allocation for the small outputs
    ints = lens.new_empty(3 * n_rows + 2 * B + 1)
    positions, slots, token_seq, q_cu, kv_lens = ints.split((n_rows, n_rows, n_rows, B + 1, B))
    out = lens.new_empty((B, max_blocks))
    tree = None if parents is None else lens.new_empty((n_rows, words), dtype=torch.int64)
    at = ints.data_ptr()
    _launch(lens.get_device(), "xl_step_rows", tables.data_ptr(), lens.data_ptr(), seqs.data_ptr(), counts.data_ptr(), _ptr(parents), at,
            at + 4 * n_rows, at + 8 * n_rows, at + 12 * n_rows, at + 12 * n_rows + 4 * B + 4, out.data_ptr(), _ptr(tree), tables.shape[0],
            tables.stride(0), B, n_rows, max_q, max_blocks, block_size, words)
    return StepRows(positions, slots, token_seq, q_cu, kv_lens, out, tree)


def tree_attention(q, k_cache, v_cache, inp, tree, scale, window) -> torch.Tensor:
    T, Hq, D = q.shape
    dev = q.get_device()
    out = q.new_empty((T, Hq * D))
    block, Hkv = k_cache.shape[1], k_cache.shape[2]
    f32, B, max_q, max_kv, sms = q.dtype is torch.float32, inp.n_seqs, inp.max_q, inp.max_kv, _sms(dev)
    # one CTA per SM, fewer where there are fewer key tiles (of 64 keys for up to 128 rows)
    ctas = max(1, min(sms, (max_kv // 64 + 1) * Hkv * (B + T * (Hq // Hkv) // 128)))
    # no tensor-core kernel: for scores that do not grow with the product, nor where the caches lie off 16-byte boundaries
    plain = f32 or scale <= 0 or B == 0 or (k_cache.data_ptr() | v_cache.data_ptr()) % 16 != 0
    size, tc = _workspace(T, B, block, Hq, Hkv, D, int(plain), max_q, max_kv, ctas, sms)
    if q.stride(2) != 1 or (tc and (q.stride(1) < 1 or q.stride(0) < 1 or q.stride(1) % 8 or q.stride(0) % max(8, q.stride(1)) or q.data_ptr() % 16)):
        q = q.contiguous()
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    bt = inp.block_tables
    _launch(dev, "xl_attention_tree", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), inp.q_cu.data_ptr(),
            inp.kv_lens.data_ptr(), bt.data_ptr(), inp.token_seq.data_ptr(), inp.positions.data_ptr(), tree.data_ptr(), T, B, bt.shape[1], block,
            k_cache.shape[0], Hq, Hkv, D, tree.shape[1], q.stride(0), q.stride(1), scale, window, int(f32), max_q, max_kv, ctas, sms, int(tc),
            _ptr(work), size)
    cuda_ops.launch_count += T > 0 and (ctas > 1 or not tc)      # the join of pieces
    return out


def adjust_logits(logits, q_cu, seqs, history, penalties, tokens, parents, bias, mask, max_q) -> torch.Tensor:
    S, V = logits.shape
    text, lens, prompts = history if history is not None else (None, None, None)
    rep, freq, pres = penalties if history is not None else (None, None, None)
    cu, ids, values = bias if bias is not None else (None, None, None)
    words, mask_of = mask if mask is not None else (None, None)
    B = q_cu.numel() - 1
    pool = lens.numel() if lens is not None else cu.numel() - 1 if cu is not None else B
    _launch(logits.get_device(), "xl_adjust_logits", logits.data_ptr(), int(logits.dtype == torch.float32), S, V, logits.stride(0), q_cu.data_ptr(),
            _ptr(seqs), B, pool, max_q, _ptr(text), 0 if text is None else text.stride(0), 0 if text is None else text.shape[1], _ptr(lens),
            _ptr(prompts), _ptr(rep), _ptr(freq), _ptr(pres), _ptr(tokens if history is not None else None), _ptr(parents), _ptr(cu), _ptr(ids),
            _ptr(values), 0 if ids is None else ids.numel(), _ptr(words), 0 if words is None else words.stride(0),
            0 if words is None else words.shape[0], _ptr(mask_of))
    return logits


def accept_tree(target, inp, parents, caches, at, depth):
    """`at`: the caches' addresses."""
    B, n, block = inp.n_seqs, len(caches), inp.block_size
    rows, blocks, all_, shape, dtype = [], [], 0, None, None
    for c, p in zip(caches, at):
        if c.shape != shape or c.dtype is not dtype:
            shape, dtype = c.shape, c.dtype
            r = c.nbytes // max(1, shape[0] * block)             # bytes of a row
        blocks.append(shape[0])
        rows.append(r)
        all_ |= p | r
    # the widest unit that divides every cache's rows and address
    unit = next(u for u in (16, 4, 2, 1) if all_ % u == 0)
    ints = target.new_empty((2 * depth + 3, B))
    out, path = ints.as_strided((B, depth + 1), (depth + 1, 1), 0), ints.as_strided((B, depth + 1), (depth + 1, 1), B * (depth + 1))
    accepted = ints[2 * depth + 2]
    to = ints.data_ptr()
    bt = inp.block_tables
    _launch(target.get_device(), "xl_accept_tree", target.data_ptr(), inp.tokens.data_ptr(), parents.data_ptr(), inp.q_cu.data_ptr(),
            inp.kv_lens.data_ptr(), bt.data_ptr(), to, to + 8 * B * (depth + 1), to + 4 * B * (depth + 1), target.numel(), B, bt.shape[1], block, depth,
            (_P * n)(*at), (_I * n)(*(rows if unit == 1 else [r // unit for r in rows])), (_I * n)(*blocks), n, unit)
    return out, accepted, path
