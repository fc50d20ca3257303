"""Greedy generation with trees of drafted tokens on a small Qwen3 through the public operators (maps from lengths, attention, rules on
logits, acceptance), against the ordinary forward pass over the text so far with the rules' definition behind it."""
import numpy as np
import torch

import oracle_tree as oracle
from helpers.paged_step import PagedStep
from xllm_wxh_b200 import ops
from xllm_wxh_b200.framework.step_input import TreeStep
from xllm_wxh_b200.models.args import ModelArgs
from xllm_wxh_b200.models.qwen import QwenForCausalLM

I32 = torch.int32
VOCAB, BLOCK, POOL, CAP = 96, 4, 5, 96


class Rules:
    """Penalties, biases and masks of the requests; the mask of a row goes by its text's length."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.penalties = (1 + torch.rand(POOL, generator=g), torch.rand(POOL, generator=g) * 0.5, torch.rand(POOL, generator=g) * 0.5)
        self.bias = (torch.arange(POOL + 1, dtype=I32) * 4, torch.randint(0, VOCAB, (POOL * 4,), generator=g, dtype=I32), torch.randn(POOL * 4, generator=g) * 2)
        self.words = torch.randint(-2 ** 31, 2 ** 31, (7, VOCAB // 32), generator=g, dtype=torch.int64).int()

    def mask_of(self, length):
        return length % 9 - 1 if length % 9 <= 7 else -1       # -1 .. 6


def plain_logits(model, text, device):
    """Logits behind every token of a text by an ordinary step over all of it."""
    a = model.args
    shape = (len(text), a.n_kv_heads, a.head_dim)
    step = PagedStep([(0, len(text))], [[torch.zeros(shape, dtype=model.dtype) for _ in range(2 * a.n_layers)]], BLOCK, device)
    step.inp.tokens.copy_(torch.tensor(text, dtype=I32))
    for c in step.caches:
        c.zero_()
    hidden = model.forward(step.inp, list(zip(step.caches[::2], step.caches[1::2])))
    return model.logits(hidden, None).float().cpu()


def ruled(row, text, prompt, p, rules):
    """The rules' definition on the logits behind `text`."""
    history = (torch.tensor([text] * POOL, dtype=I32), torch.full((POOL,), len(text), dtype=I32), torch.full((POOL,), prompt, dtype=I32))
    mask = (rules.words, torch.tensor([rules.mask_of(len(text))], dtype=I32))
    return oracle.logits(row[None], [0, 1], [p], history, rules.penalties, None, None, rules.bias, mask)[0][0]


def plain_generation(model, prompts, seqs, rules, n_new, device):
    texts = []
    for prompt, p in zip(prompts, seqs):
        text = list(prompt)
        for _ in range(n_new):
            text.append(int(ruled(plain_logits(model, text, device)[-1], text, len(prompt), p, rules).argmax()))
        texts.append(text)
    return texts


def drafted_generation(model, prompts, seqs, rules, n_new, device, guesses, seed=0):
    """`guesses[b]`: a text whose continuation the drafts mostly propose.  Returns the texts, the ruled logits that every token came from,
    and how many drafted tokens were accepted."""
    rng = np.random.default_rng(seed)
    B, MB = len(prompts), -(-CAP // BLOCK)
    dev = lambda t: t.to(device)
    a = model.args
    tables = dev((torch.from_numpy(rng.permutation(POOL * MB).astype(np.int32)) + 1).view(POOL, MB))
    caches = [torch.zeros(POOL * MB + 1, BLOCK, a.n_kv_heads, a.head_dim, dtype=model.dtype, device=device) for _ in range(2 * a.n_layers)]
    kv = list(zip(caches[::2], caches[1::2]))
    lens, history = torch.zeros(POOL, dtype=I32, device=device), torch.zeros(POOL, CAP, dtype=I32, device=device)
    prompt_lens = torch.zeros(POOL, dtype=I32)
    for b, p in enumerate(seqs):
        prompt_lens[p] = len(prompts[b])
    prompt_lens, seq_ids = dev(prompt_lens), dev(torch.tensor(seqs, dtype=I32))
    penalties, bias, words = tuple(dev(t) for t in rules.penalties), tuple(dev(t) for t in rules.bias), dev(rules.words)

    def step(rows, parents):
        n_rows, most = sum(map(len, rows)) + 3, max(map(len, rows))
        flat = dev(torch.tensor([t for r in rows for t in r] + [0] * 3, dtype=I32))
        up = dev(torch.tensor([t for r in parents for t in r] + [0] * 3, dtype=I32))
        counts = dev(torch.tensor([len(r) for r in rows], dtype=I32))
        maps = ops.step_rows(tables, lens, seq_ids, counts, n_rows, BLOCK, up, max_q=most)
        inp = TreeStep(flat, maps, BLOCK, most, CAP)
        return inp, up, model.logits(model.forward(inp, kv), None)

    texts = [list(p) for p in prompts]
    step([p[:-1] for p in prompts], [list(range(-1, len(p) - 2)) for p in prompts])
    for b, p in enumerate(seqs):
        history[p, :len(prompts[b]) - 1] = dev(torch.tensor(prompts[b][:-1], dtype=I32))
        lens[p] = len(prompts[b]) - 1
    seen, agreed = [[] for _ in prompts], 0
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < n_new:
        rows, parents = [], []
        for b, text in enumerate(texts):
            row, up, spine = [text[-1]], [-1], 0
            ahead = guesses[b][len(text):len(text) + 3]
            for t in ahead:
                for wrong in rng.integers(0, VOCAB, rng.integers(0, 3)).tolist():
                    row.append(wrong)
                    up.append(spine)
                row.append(t if rng.random() < 0.9 else (t + 1) % VOCAB)
                up.append(spine)
                spine = len(row) - 1
            rows.append(row)
            parents.append(up)
        inp, up, logits = step(rows, parents)
        base = [len(t) - 1 for t in texts]
        of = [rules.mask_of(base[b] + len(oracle.line(parents[b], i))) for b, r in enumerate(rows) for i in range(len(r))]
        mask = (words, dev(torch.tensor(of + [-1] * 3, dtype=I32)))
        ops.adjust_logits(logits, inp.q_cu, seq_ids, (history, lens, prompt_lens), penalties, inp.tokens, up, bias, mask, max_q=inp.max_q)
        target = logits.float().argmax(-1).int()
        out, accepted, path = ops.accept_tree(target, inp, up, caches)
        cu = inp.q_cu.tolist()
        for b, p in enumerate(seqs):
            got = [t for t in out[b].tolist() if t >= 0]
            agreed += int(accepted[b])
            for r in path[b].tolist()[:len(got)]:
                seen[b].append(logits[cu[b] + r].float().cpu())
            history[p, base[b]:base[b] + len(got)] = dev(torch.tensor([texts[b][-1]] + got[:-1], dtype=I32))
            texts[b] += got
            lens[p] += len(got)
    return texts, seen, agreed


def check_generation(device, dtype):
    args = ModelArgs(model_type="qwen3", vocab_size=VOCAB, hidden_size=128, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, intermediate_size=160,
                     qk_norm=True, max_position_embeddings=512)
    model = QwenForCausalLM(args, None, device, dtype)
    model.init_random(3)
    if hasattr(model, "finalize_weights"):
        model.finalize_weights()
    rng, rules, n_new, seqs = np.random.default_rng(4), Rules(5), 14, [3, 0, 4]
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (9, 2, 21)]
    with torch.inference_mode():
        plain = plain_generation(model, prompts, seqs, rules, n_new, device)
        texts, seen, agreed = drafted_generation(model, prompts, seqs, rules, n_new, device, plain)
        for b, (text, p) in enumerate(zip(texts, seqs)):
            n = len(prompts[b])
            if dtype == torch.float32:
                assert text[:n + n_new] == plain[b][:n + n_new]
            # each token's logits are those of an ordinary pass over the text in front of it
            rows = plain_logits(model, text, device)
            for i, got in enumerate(seen[b]):
                want = ruled(rows[n - 1 + i], text[:n + i], n, p, rules)
                open_ = want != -float("inf")
                assert torch.equal(open_, got != -float("inf")) and text[n + i] == int(got.argmax())
                # two layers of bf16 roundings (2^-9 on average, some thirty in a row, adding like a random walk) stay below a few percent
                assert (got.double() - want)[open_].norm() <= (0.05 if dtype == torch.bfloat16 else 1e-4) * want[open_].norm()
        assert agreed > 10
