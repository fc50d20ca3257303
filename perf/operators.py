"""Cases of the operators that a serving step with drafted token trees runs, their plain forms and their definitions in 64 bits.

A sequence's drafted tokens form a tree: row 0 is the token emitted last, every other row follows the row `parents` names.  One step of
such sequences builds its maps on the device from the lengths (`step_rows`), attends to the cache and to each row's own ancestors
(`tree_attention`), applies penalties, biases and grammar masks to the logits of every row (`adjust_logits`), and keeps the path that the
target model agrees with (`accept_tree`).
"""
import math
import types

import torch

own = False

I32, I64, F32 = torch.int32, torch.int64, torch.float32
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one user, a small tree: nothing but latency counts
        rows_case("rows: 1 sequence, 8 nodes", 1, 8, 256, 16, 1, 3000, tree=True),
        # a chain of single drafted tokens over a full batch of 32k-token tables in blocks of 16; an eighth of the places are padding
        rows_case("rows: 256 sequences, single rows", 256, 1, 2048, 16, 1, 32000, tree=False, pad=32),
        # a large batch of trees with tables for 128k tokens in blocks of 16
        rows_case("rows: 1024 trees of 32", 1024, 32, 8192, 16, 100, 130000, tree=True),
        # one user behind a prompt of a thousand tokens: a tree of 16 nodes, 8 key heads for 32 query heads, default block size
        attention_case("attention: 1 x 16, context 1000", 1, 16, 16, 1000, 1000, 32, 8, 128, 128, "bf16"),
        # a batch in full swing: ragged contexts, trees of 9 to 32 nodes
        attention_case("attention: 64 x 32, context to 8192", 64, 9, 32, 300, 8192, 32, 8, 128, 128, "bf16"),
        # long contexts, 64 nodes for 8 query heads per key head: products and exponentials count as much as bytes
        attention_case("attention: 16 x 64, context to 32768", 16, 64, 64, 16000, 32704, 64, 8, 128, 128, "bf16"),
        # 7 query heads per key head, 64 columns, blocks of 16, a sliding window, trees of 1 to 25 nodes, some sequences without a past
        attention_case("attention: 24 x 25, 28/4 heads, window", 24, 1, 25, 0, 3001, 28, 4, 64, 16, "bf16", window=1500),
        # a model in true 32-bit
        attention_case("attention: 8 x 12 in 32-bit", 8, 3, 12, 50, 2000, 14, 2, 64, 16, "f32"),
        # a decoding batch: 2 to 3 thousand tokens of history, biases on some ids, a grammar for every fourth request
        logits_case("logits: 256 rows, history to 3100", 256, 1, 1, 151936, 50, 3100, 40, 64, "bf16"),
        # trees under a grammar: 16 rows for each of 64 requests, a mask for every row
        logits_case("logits: 64 x 16 rows, all masked", 64, 16, 16, 152064, 200, 8000, 300, 1024, "f32"),
        # one user, two layers
        accept_case("accept: 1 x 8, 2 layers", 1, 8, 8, 2, 2, 64, 16, 500, "bf16"),
        # a batch of trees, the caches of 36 layers
        accept_case("accept: 64 x 32, 36 layers", 64, 9, 32, 36, 8, 128, 16, 90, "bf16"),
    ]


def rows_case(name, seqs, nodes, blocks, block, lo, hi, tree, pad=0):
    return dict(name=name, op="rows", seqs=seqs, nodes_lo=nodes, nodes=nodes, blocks=blocks, block=block, lo=lo, hi=hi, tree=tree, pad=pad)


def attention_case(name, seqs, nodes_lo, nodes, lo, hi, heads, kv_heads, dim, block, dtype, window=-1):
    return dict(name=name, op="attention", seqs=seqs, nodes_lo=nodes_lo, nodes=nodes, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim,
                block=block, dtype=dtype, window=window)


def logits_case(name, seqs, nodes_lo, nodes, vocab, lo, hi, biases, masks, dtype):
    return dict(name=name, op="logits", seqs=seqs, nodes_lo=nodes_lo, nodes=nodes, vocab=vocab, lo=lo, hi=hi, biases=biases, masks=masks, dtype=dtype)


def accept_case(name, seqs, nodes_lo, nodes, layers, kv_heads, dim, block, hi, dtype):
    return dict(name=name, op="accept", seqs=seqs, nodes_lo=nodes_lo, nodes=nodes, layers=layers, kv_heads=kv_heads, dim=dim, block=block,
                lo=0, hi=hi, dtype=dtype)


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    op = rng.choice(["rows", "attention", "attention", "logits", "accept"])
    nodes = log(1, 64)
    nodes_lo = rng.randint(1, nodes)
    if op == "rows":
        block, tree = rng.choice([8, 16, 32, 128]), rng.random() < 0.6
        blocks = log(16, 8192)
        seqs = min(log(1, 1024), (1024 * 8192) // blocks)
        nodes = nodes if tree else log(1, 2000)
        nodes = min(nodes, 32 * 1024 // seqs, block * blocks // 2)
        hi = block * blocks - nodes - 1
        c = rows_case("", seqs, nodes, blocks, block, rng.randint(0, hi // 2), hi, tree, rng.choice([0, seqs // 8]))
        c["nodes_lo"] = rng.randint(0, nodes)
    elif op == "attention":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 4), (28, 4), (40, 8), (8, 8), (16, 2), (14, 2)])
        dim = rng.choice([64, 128, 128])
        seqs, hi = log(1, 128), log(1, 32000)
        if dtype == "f32":
            seqs, hi, nodes = min(seqs, 16), min(hi, 2500), min(nodes, 16)
        while seqs * nodes * heads * hi > 16 * 64 * 64 * 16000 or seqs * kv_heads * hi * dim > 16 * 8 * 24000 * 128:
            seqs, hi = (seqs + 1) // 2, (hi + 1) // 2
        c = attention_case("", seqs, min(nodes_lo, nodes), nodes, rng.randint(0, hi), hi, heads, kv_heads, dim, rng.choice([16, 32, 64, 128]), dtype,
                           rng.choice([-1, -1, 1000]))
    elif op == "logits":
        vocab = rng.choice([32000, 151936, 152064, 128257, 4099])
        seqs, hi, nodes = log(1, 256), log(1, 12000), min(nodes, 32)
        while seqs * nodes > 1024:
            seqs, nodes = (seqs + 1) // 2, (nodes + 1) // 2
        c = logits_case("", seqs, min(nodes_lo, nodes), nodes, vocab, rng.randint(0, hi), hi, rng.choice([0, 5, 300]), rng.randint(0, seqs * nodes),
                        rng.choice(["bf16", "f32"]))
    else:
        dtype = rng.choice(["bf16", "bf16", "f32"])
        seqs, layers = log(1, 64), log(1, 36 if dtype == "bf16" else 16)
        c = accept_case("", seqs, min(nodes_lo, 32), min(nodes, 32), layers, rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32]),
                        rng.randint(1, 90), dtype)
    c.pop("name")
    return c


# ----------------------------------------------------------------------------- inputs
def spread(lo, hi, n):
    """n whole numbers from lo to hi at even distances: ragged, with a known sum."""
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def lens_of(c):
    return spread(c["lo"], c["hi"], c["seqs"])


def counts_of(c):
    return spread(c["nodes_lo"], c["nodes"], c["seqs"])


class Draws:
    """Random inputs of one seed, on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda").manual_seed(seed)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=I32)

    def unit(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def normal(self, *shape, dtype=F32):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda", dtype=I32)

    def shuffled(self, values):
        t = torch.tensor(values, device="cuda", dtype=I32)
        return t[self.perm(len(values)).long()]


def ragged(counts, total):
    """(q_cu [B + 1], sequence of each row, number of the row in its sequence); `total` is the sum of counts."""
    q_cu = torch.zeros(counts.numel() + 1, device="cuda", dtype=I64)
    q_cu[1:] = counts.long().cumsum(0)
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device="cuda"), counts.long(), output_size=total)
    return q_cu, seq, torch.arange(total, device="cuda") - q_cu[seq]


def random_parents(d, at):
    """A random tree for every sequence: row 0 is the root, row i follows one of the rows before it, early rows more often."""
    p = (d.unit(at.numel()) ** 1.5 * at).floor().to(I32)
    return torch.where(at == 0, torch.full_like(p, -1), torch.minimum(p, (at - 1).to(I32)))


def prepare(case, seed):
    d, c = Draws(seed), dict(case)
    s = types.SimpleNamespace(case=c)
    B, N = c["seqs"], c["nodes"]
    counts = d.shuffled(counts_of(c))
    total = sum(counts_of(c))
    if c["op"] == "rows":
        pool = B + 3
        s.tables = d.ints(1, 1 << 20, pool, c["blocks"])
        lens = d.ints(0, c["lo"] + 1, pool)
        s.seqs = d.perm(pool)[:B].clone()
        lens[s.seqs.long()] = d.shuffled(lens_of(c))
        s.lens = lens
        if c["pad"]:                                   # places of a full batch that hold no sequence
            s.seqs[B - c["pad"]:] = -1
        s.counts, s.n_rows = counts, -(-total // 64) * 64
        live = torch.where(s.seqs >= 0, counts, torch.zeros_like(counts))
        s.total = int(live.sum())
        s.parents = None
        if c["tree"]:
            s.parents = torch.zeros(s.n_rows, device="cuda", dtype=I32)
            s.parents[:s.total] = random_parents(d, ragged(live, s.total)[2])
        return s
    q_cu, seq, at = ragged(counts, total)
    parents = random_parents(d, at)
    if c["op"] == "logits":
        V = c["vocab"]
        zipf = lambda *shape: (float(V) ** d.unit(*shape)).long().clamp(1, V).to(I32) - 1      # small ids are common, as in text
        s.logits = (d.normal(total, V) * 3).to(TYPES[c["dtype"]])
        s.q_cu, s.parents, s.tokens, s.max_q = q_cu.to(I32), parents, zipf(total), N
        pool = B + 2
        s.seqs = d.perm(pool)[:B].clone()
        s.text, s.lens = zipf(pool, c["hi"] + 1), torch.zeros(pool, device="cuda", dtype=I32)
        s.lens[s.seqs.long()] = d.shuffled(lens_of(c))
        s.prompts = (s.lens * d.unit(pool)).to(I32)
        some = lambda x: torch.where(d.unit(pool) < 0.25, torch.zeros_like(x), x)                   # a quarter of the requests ask for none
        s.rep, s.freq, s.pres = 1 + some(d.unit(pool) * 0.3), some(d.unit(pool) - 0.3), some(d.unit(pool) - 0.3)
        s.bias = None
        if c["biases"]:
            n = d.shuffled(spread(0, c["biases"], pool))
            cu = torch.zeros(pool + 1, device="cuda", dtype=I32)
            cu[1:] = n.cumsum(0)
            m = sum(spread(0, c["biases"], pool))
            s.bias = (cu, d.ints(0, V, m), d.normal(m) * 5)
        s.mask = None
        if c["masks"]:
            M, W = c["masks"], -(-V // 32)
            words = d.ints(-2 ** 31, 2 ** 31 - 1, M, W)
            tight = words & d.ints(-2 ** 31, 2 ** 31 - 1, M, W) & d.ints(-2 ** 31, 2 ** 31 - 1, M, W) & d.ints(-2 ** 31, 2 ** 31 - 1, M, W)
            tight = torch.where(d.unit(M, W) < 0.1, tight, torch.zeros_like(tight))               # a few allowed tokens
            loose = torch.where(d.unit(M, W) < 0.05, words, torch.full_like(words, -1))           # a few forbidden ones
            of = torch.full((total,), -1, device="cuda", dtype=I32)
            of[d.perm(total).long()[:M]] = d.perm(M)[:total]
            s.mask = (torch.where(d.unit(M, 1) < 0.7, tight, loose), of)
        return s
    lens = d.shuffled(lens_of(c))
    block = c["block"]
    need = [-(-(x + N) // block) for x in lens_of(c)]
    MB, blocks = max(need), sum(need) + 1
    dtype, kv, dim = TYPES[c["dtype"]], c["kv_heads"], c["dim"]
    # every sequence's blocks lie anywhere in the cache; table entries past its last block are 0
    held = (lens + N + block - 1) // block
    first = held.cumsum(0) - held
    ids = d.perm(blocks - 1) + 1
    place = torch.arange(MB, device="cuda")[None]
    tables = torch.where(place < held[:, None], ids[(first[:, None] + place).clamp(max=blocks - 2).long()], torch.zeros(1, device="cuda", dtype=I32))
    anc = ancestors(parents, seq, at, B, N)
    st = types.SimpleNamespace(q_cu=q_cu.to(I32), kv_lens=lens + counts, block_tables=tables.contiguous(), token_seq=seq.to(I32), n_seqs=B,
                               positions=(lens[seq] + anc.sum(-1)[seq, at] - 1).to(I32), max_q=N, max_kv=c["hi"] + N, block_size=block)
    s.step, s.parents, s.lens = st, parents, lens
    if c["op"] == "attention":
        H = c["heads"]
        st.tree = pack(anc)[seq, at]
        qkv = d.normal(total, (H + 2 * kv) * dim, dtype=dtype)
        qkv[:, :H * dim] *= 2
        s.q = qkv[:, :H * dim].view(total, H, dim)                     # a view of the projection's rows, as a model has it
        s.k, s.v = d.normal(blocks, block, kv, dim, dtype=dtype), d.normal(blocks, block, kv, dim, dtype=dtype)
        return s
    st.tokens = d.ints(0, 50000, total)
    # the target model agrees with one child of most rows
    child = torch.full((total,), -1, device="cuda", dtype=I64)
    up = q_cu[seq] + parents.clamp(min=0)
    child.scatter_reduce_(0, torch.where(parents >= 0, up, torch.arange(total, device="cuda")),
                          torch.where(parents >= 0, torch.arange(total, device="cuda"), child), "amax")
    agree = (child >= 0) & (d.unit(total) < 0.8)
    s.target = torch.where(agree, st.tokens[child.clamp(min=0)], d.ints(0, 50000, total))
    s.caches = d.normal(2 * c["layers"], blocks, block, kv, dim, dtype=dtype)
    s.depth = N - 1
    return s


# ----------------------------------------------------------------------------- plain forms
def ancestors(parents, seq, at, B, N):
    """[B, N, N] truth values: row i of a sequence is row j or follows it (closure of the parents by squaring)."""
    a = torch.zeros(B, N, N, device="cuda")
    a[seq, at, at] = 1
    has = parents >= 0
    a[seq[has], at[has], parents[has].long()] = 1
    return closure(a, N) > 0


def closure(a, n):
    return a if n <= 1 else closure((a @ a > 0).float(), (n + 1) // 2)


def pack(anc):
    """Bits of 64 rows to a word."""
    B, N, _ = anc.shape
    W = -(-N // 64)
    a = torch.zeros(B, N, W * 64, device="cuda", dtype=I64)
    a[..., :N] = anc
    return (a.view(B, N, W, 64) << torch.arange(64, device="cuda")).sum(-1)


def run(state):
    return {"rows": run_rows, "attention": run_attention, "logits": run_logits, "accept": run_accept}[state.case["op"]](state)


def run_rows(s):
    c = s.case
    if own:
        from xllm_wxh_b200 import ops
        return tuple(ops.step_rows(s.tables, s.lens, s.seqs, s.counts, s.n_rows, c["block"], s.parents, max_q=max(1, c["nodes"])))
    B, T, block, MB = c["seqs"], s.n_rows, c["block"], c["blocks"]
    live = s.seqs >= 0
    pool = s.seqs.clamp(min=0).long()
    counts = torch.where(live, s.counts, torch.zeros_like(s.counts))
    before = torch.where(live, s.lens[pool], torch.zeros_like(s.counts))
    q_cu = torch.zeros(B + 1, device="cuda", dtype=I64)
    q_cu[1:] = counts.cumsum(0)
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(q_cu[1:], t, right=True)
    pad = seq >= B
    sq = seq.clamp(max=B - 1)
    at = t - q_cu[sq]
    kv = before + counts
    place = torch.arange(MB, device="cuda")[None]
    tables = torch.where(place < ((kv + block - 1) // block)[:, None], s.tables[pool], torch.zeros(1, device="cuda", dtype=I32))
    p = before[sq] + at
    slots = torch.where(pad, t % block, s.tables[pool[sq], torch.where(pad, 0, p // block)].long() * block + p % block)
    tree, depth = None, at
    if s.parents is not None:
        N = max(1, c["nodes"])
        real = ~pad
        anc = ancestors(s.parents[real], seq[real], at[real], B, N)
        words = pack(anc)
        rank = at.clamp(0, N - 1)
        tree = torch.where(pad[:, None], torch.zeros(1, device="cuda", dtype=I64), words[sq, rank])
        depth = anc.sum(-1)[sq, rank] - 1
    positions = torch.where(pad, 0, before[sq] + depth)
    return positions.to(I32), slots.to(I32), torch.where(pad, -1, seq).to(I32), q_cu.to(I32), kv.to(I32), tables, tree


def visible(s, N, L):
    """[B, N, L] truth values: what each row may see (rows past a sequence's last see nothing)."""
    c, st = s.case, s.step
    B = c["seqs"]
    counts = st.q_cu.diff().long()
    row = torch.arange(N, device="cuda")[None]
    real = row < counts[:, None]
    t = (st.q_cu[:-1].long()[:, None] + row).clamp(max=st.token_seq.numel() - 1)
    base = st.kv_lens.long() - counts
    key = torch.arange(L, device="cuda")[None]
    node = key - base[:, None]                                          # number of the key among the sequence's rows
    isnode = (node >= 0) & (node < counts[:, None])
    n = node.clamp(0, N - 1)
    word = st.tree[t][torch.arange(B, device="cuda")[:, None, None], torch.arange(N, device="cuda")[None, :, None], (n // 64)[:, None, :]]
    bit = (word >> (n % 64)[:, None, :]) & 1
    see = torch.where(isnode[:, None], bit > 0, (key < base[:, None])[:, None])
    if c["window"] > 0:
        pos = st.positions[t].long()
        of_key = torch.where(isnode, pos.gather(1, n), key.expand(B, L))
        see = see & (of_key[:, None, :] > pos[:, :, None] - c["window"])
    return see & real[..., None], t, real


def run_attention(s):
    c, st = s.case, s.step
    H, kv, D, B, N = c["heads"], c["kv_heads"], c["dim"], c["seqs"], c["nodes"]
    scale = D ** -0.5
    if own:
        from xllm_wxh_b200 import ops
        return ops.tree_attention(s.q, s.k, s.v, st, st.tree, scale, c["window"])
    MB = st.block_tables.shape[1]
    L = MB * c["block"]
    see, t, real = visible(s, N, L)
    k = s.k[st.block_tables.long()].view(B, L, kv, D).permute(0, 2, 3, 1).float()
    q = s.q[t].float().view(B, N, kv, H // kv, D).permute(0, 2, 3, 1, 4).reshape(B, kv, H // kv * N, D)
    x = ((q @ k) * scale).view(B, kv, H // kv, N, L).masked_fill_(~see[:, None, None], -math.inf)
    del k, q
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = s.v[st.block_tables.long()].view(B, L, kv, D).transpose(1, 2).float()
    o = (x.view(B, kv, H // kv * N, L) @ v).view(B, kv, H // kv, N, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(B, N, H * D)
    return o[real].to(s.q.dtype)


def run_logits(s):
    c = s.case
    if own:
        from xllm_wxh_b200 import ops
        return ops.adjust_logits(s.logits, s.q_cu, s.seqs, (s.text, s.lens, s.prompts), (s.rep, s.freq, s.pres), s.tokens, s.parents, s.bias, s.mask,
                                 s.max_q)
    B, V, N, S = c["seqs"], c["vocab"], c["nodes"], s.logits.shape[0]
    q_cu, seq, at = ragged(s.q_cu.diff(), S)
    pool = s.seqs.long()
    text = s.text[pool].long()
    place = torch.arange(text.shape[1], device="cuda")[None]
    there = place < s.lens[pool][:, None]
    seen = torch.zeros(B, V, device="cuda").scatter_add_(1, text, there.float())
    made = torch.zeros(B, V, device="cuda").scatter_add_(1, text, (there & (place >= s.prompts[pool][:, None])).float())
    anc = ancestors(s.parents, seq, at, B, N)[seq, at]                     # [S, N]
    node = (q_cu[seq][:, None] + torch.arange(N, device="cuda")).clamp(max=S - 1)
    path = torch.zeros(S, V, device="cuda").scatter_add_(1, s.tokens[node].long(), anc.float())
    made = made[seq] + path
    seen = seen[seq] + path
    p = pool[seq]
    x = s.logits.float()
    y = x - made * s.freq[p][:, None] - (made > 0) * s.pres[p][:, None]
    y = torch.where(y < 0, y * s.rep[p][:, None], y / s.rep[p][:, None])
    x = torch.where(seen > 0, y, x)
    if s.bias is not None:
        cu, ids, values = s.bias
        e = torch.arange(ids.numel(), device="cuda")
        owner = torch.searchsorted(cu[1:].long(), e, right=True)
        last = torch.full(((cu.numel() - 1) * V,), -1, device="cuda", dtype=I64).scatter_reduce_(0, owner * V + ids.long(), e, "amax").view(-1, V)
        dense = torch.where(last >= 0, values[last.clamp(min=0)], torch.zeros(1, device="cuda"))
        x = x + dense[p]
    if s.mask is not None:
        words, of = s.mask
        id_ = torch.arange(V, device="cuda")
        m = of.clamp(min=0).long()
        bits = (words[m][:, id_ // 32] >> (id_ % 32).to(I32)[None]) & 1
        x = x.masked_fill_((bits == 0) & (of >= 0)[:, None], -math.inf)
    return s.logits.copy_(x)


def run_accept(s):
    c, st = s.case, s.step
    if own:
        from xllm_wxh_b200 import ops
        return (*ops.accept_tree(s.target, st, s.parents, list(s.caches), s.depth), s.caches)
    B, N, block, T = c["seqs"], c["nodes"], c["block"], s.target.numel()
    q_cu, seq, at = ragged(st.q_cu.diff(), T)
    row = torch.arange(N, device="cuda")[None]
    t = (q_cu[:-1, None] + row).clamp(max=T - 1)
    real = row < st.q_cu.diff()[:, None]
    up = s.parents[t].long()
    agrees = real & (up >= 0) & (st.tokens[t] == s.target[t].gather(1, up.clamp(min=0)))
    # of several children that agree, the first one counts
    twin = agrees[:, :, None] & agrees[:, None, :] & (up[:, :, None] == up[:, None, :]) & (row[0][None, :] < row[0][:, None])
    kept = (agrees & ~twin.any(-1)) | (real & (row == 0))
    anc = ancestors(s.parents, seq, at, B, N)
    on = real & ~(anc & ~kept[:, None, :]).any(-1)
    depth = torch.where(on, anc.sum(-1) - 1, N)                            # rows off the path go to a column that is cut off
    out = torch.full((B, N + 1), -1, device="cuda", dtype=I32).scatter_(1, depth, s.target[t])[:, :N]
    path = torch.full((B, N + 1), -1, device="cuda", dtype=I32).scatter_(1, depth, row.expand(B, N).to(I32))[:, :N]
    base = st.kv_lens.long() - st.q_cu.diff()
    slot = lambda p: st.block_tables.gather(1, p // block).long() * block + p % block
    move = path >= 0
    src, dst = slot(base[:, None] + path.clamp(min=0))[move], slot(base[:, None] + row)[move]
    flat = s.caches.view(2 * c["layers"], -1, c["kv_heads"], c["dim"])
    flat[:, dst] = flat[:, src]
    return out, (move.sum(1) - 1).to(I32), path, s.caches


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    B, lens, counts = c["seqs"], lens_of(c), counts_of(c)
    T, size = sum(counts), 2 if c.get("dtype") == "bf16" else 4
    if c["op"] == "rows":
        used = sum(-(-(a + b) // c["block"]) for a, b in zip(lens, counts)) * (B - c["pad"]) // max(1, B)
        rows = -(-T // 64) * 64
        return {"bytes": 4 * (used + B * c["blocks"] + 4 * B + 3 * rows) + (rows * (4 + 8 * -(-max(1, c["nodes"]) // 64)) if c["tree"] else 0), "flops": 10 * rows}
    if c["op"] == "attention":
        H, kv, D, w = c["heads"], c["kv_heads"], c["dim"], c["window"]
        keys = [min(a + b, w + b) if w > 0 else a + b for a, b in zip(lens, counts)]
        return {"bytes": size * D * (2 * kv * sum(keys) + 2 * H * T) + 8 * T, "flops": 4 * D * H * sum(k * n for k, n in zip(keys, counts))}
    if c["op"] == "logits":
        # ids of the histories; every logit that a penalty or a bias changes (at most the distinct ids: about a third of the text) read and
        # written; forbidden logits written; masks read
        touched = sum(n * (0.35 * a + n + c["biases"] / 2) for a, n in zip(lens, counts))
        masks = min(c["masks"], T)
        return {"bytes": 4 * sum(lens) + 2 * size * touched + masks * c["vocab"] * (0.7 * size + 1 / 8), "flops": 6 * touched}
    moved = 3 * B if T > B else 0                                            # about three drafted rows of a sequence are kept, most of them elsewhere
    row = size * c["kv_heads"] * c["dim"]
    return {"bytes": 12 * T + 8 * B * c["nodes"] + 2 * moved * 2 * c["layers"] * row, "flops": 4 * T}


# ----------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "rows":
        return None
    s = prepare(case, seed)
    if c["op"] == "logits":
        return exact_logits(s)
    return exact_attention(s) if c["op"] == "attention" else exact_accept(s)


def lines(s, q_cu, parents):
    """For each row of the step the rows of its sequence from itself up to the root (numbers within the sequence)."""
    found = []
    for a, b in zip(q_cu[:-1], q_cu[1:]):
        for i in range(b - a):
            line, j = [], i
            while j >= 0:
                line.append(j)
                j = parents[a + j]
            found.append(line)
    return found


def exact_attention(s):
    c, st = s.case, s.step
    H, kv, D, w = c["heads"], c["kv_heads"], c["dim"], c["window"]
    q_cu, kv_lens, parents, pos = st.q_cu.tolist(), st.kv_lens.tolist(), s.parents.tolist(), st.positions.tolist()
    line = lines(s, q_cu, parents)
    out = []
    for b in range(c["seqs"]):
        a, n = q_cu[b], q_cu[b + 1] - q_cu[b]
        L = kv_lens[b]
        ids = st.block_tables[b, :-(-L // c["block"])].long()
        see = torch.zeros(n, L, dtype=torch.bool)
        see[:, :L - n] = True
        where = list(range(L - n)) + pos[a:a + n]
        for i in range(n):
            see[i, [L - n + j for j in line[a + i]]] = True
            if w > 0:
                see[i] &= torch.tensor(where) > pos[a + i] - w
        see = see.cuda()
        for h in range(kv):
            k, v = (x[ids, :, h].reshape(-1, D)[:L].double() for x in (s.k, s.v))
            q = s.q[a:a + n, h * (H // kv):(h + 1) * (H // kv)].double()
            x = torch.einsum("ngd,ld->ngl", q, k) / math.sqrt(D)
            x.masked_fill_(~see[:, None], -math.inf)
            e = (x - x.amax(-1, keepdim=True)).exp()
            out.append((a, h, torch.einsum("ngl,ld->ngd", e / e.sum(-1, keepdim=True), v)))
    full = torch.zeros(s.q.shape[0], kv, H // kv * D, device="cuda", dtype=torch.float64)
    for a, h, o in out:
        full[a:a + o.shape[0], h] = o.reshape(o.shape[0], -1)
    return full.reshape(s.q.shape[0], H * D)


def exact_logits(s):
    c = s.case
    q_cu, parents, tokens = s.q_cu.tolist(), s.parents.tolist(), s.tokens.tolist()
    line, V = lines(s, q_cu, parents), c["vocab"]
    seqs, lens, prompts = s.seqs.tolist(), s.lens.tolist(), s.prompts.tolist()
    out = s.logits.double()
    words, of = (s.mask[0].cpu(), s.mask[1].tolist()) if s.mask is not None else (None, [-1] * len(line))
    for b, p in enumerate(seqs):
        text = s.text[p, :lens[p]].long()
        seen, made = torch.bincount(text, minlength=V), torch.bincount(text[prompts[p]:], minlength=V)
        add = torch.zeros(V, dtype=torch.float64)
        if s.bias is not None:
            lo, hi = int(s.bias[0][p]), int(s.bias[0][p + 1])
            for i, v in zip(s.bias[1][lo:hi].tolist(), s.bias[2][lo:hi].double().tolist()):
                add[i] = v
        add = add.cuda()
        rep, freq, pres = (float(t[p].double()) for t in (s.rep, s.freq, s.pres))
        for r in range(q_cu[b], q_cu[b + 1]):
            path = torch.bincount(torch.tensor([tokens[q_cu[b] + j] for j in line[r]], device="cuda"), minlength=V)
            n = (made + path).double()
            y = out[r] - n * freq - (n > 0).double() * pres
            y = torch.where(y < 0, y * rep, y / rep)
            out[r] = torch.where(seen + path > 0, y, out[r]) + add
            if of[r] >= 0:
                w = words[of[r]].to(I64).cuda() & 0xFFFFFFFF
                allowed = torch.stack([(w >> k) & 1 for k in range(32)], 1).reshape(-1)[:V]
                out[r, allowed == 0] = -math.inf
    return out


def exact_accept(s):
    c, st = s.case, s.step
    q_cu, kv_lens, parents, tokens, target, tables = (x.tolist() for x in (st.q_cu, st.kv_lens, s.parents, st.tokens, s.target, st.block_tables))
    caches, block = s.caches.clone(), c["block"]
    out, accepted, path = [], [], []
    for b in range(c["seqs"]):
        a, n = q_cu[b], q_cu[b + 1] - q_cu[b]
        at, rows = 0, [0]
        while True:
            nxt = [j for j in range(n) if parents[a + j] == at and tokens[a + j] == target[a + at]]
            if not nxt:
                break
            at = nxt[0]
            rows.append(at)
        base = kv_lens[b] - n
        place = lambda p: (tables[b][p // block], p % block)
        for i, j in enumerate(rows):
            (b0, o0), (b1, o1) = place(base + j), place(base + i)
            caches[:, b1, o1] = s.caches[:, b0, o0]
        pad = [-1] * (c["nodes"] - len(rows))
        out.append([target[a + j] for j in rows] + pad)
        path.append(rows + pad)
        accepted.append(len(rows) - 1)
    return torch.tensor(out, dtype=I32), torch.tensor(accepted, dtype=I32), torch.tensor(path, dtype=I32), caches
