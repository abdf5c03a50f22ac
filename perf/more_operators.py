"""The operators of a step that verifies drafted tokens over a shared paged cache
and what they are timed on: the tables of scaled rotary positions
(``rope_tables``), the norms of q and k heads with their rotation and the write
into pages (``rope_append``), the attention of a tree of drafted tokens
(``paged_attention`` with a plan that knows the trees), penalties, biases and
grammar masks on the nodes' logits (``adjust_logits``), and the accepted path
kept in the pages (``PagedKVCache.keep``).

Shapes are the repository's own (32q/8kv, 64q/8kv, 28q/4kv and 32q/32kv heads,
head_dim 128 or 64, 16-token pages and larger ones, contexts up to 131072
tokens, a vocabulary of 128256) or generic.
"""
import math
import random

import torch

own = False

HEADS = ((32, 8), (32, 8), (64, 8), (28, 4), (32, 32), (16, 8), (12, 1))
EPS = 1e-6


def listed():
    return [
        # a tree of eight drafts behind one user's short chat: the smallest attention call, latency bound
        {"name": "tree_small", "kind": "tree", "prompts": 1, "samples": 1, "plo": 0, "phi": 0, "olo": 1000, "ohi": 1000,
         "tlo": 8, "thi": 8, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 1, "dtype": "bf16"},
        # continuous batching with trees of 25 drafts, every sequence at its own length
        {"name": "tree_batch", "kind": "tree", "prompts": 16, "samples": 1, "plo": 0, "phi": 0, "olo": 1000,
         "ohi": 20000, "tlo": 25, "thi": 25, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 2, "dtype": "bf16"},
        # samples of two prompts, ragged trees, seven heads per KV head, head_dim 64
        {"name": "tree_prompts_f16", "kind": "tree", "prompts": 2, "samples": 6, "plo": 6000, "phi": 9001, "olo": 30,
         "ohi": 900, "tlo": 5, "thi": 31, "H": 28, "KVH": 4, "D": 64, "page": 32, "lens": 3, "dtype": "f16"},
        # the largest: wide trees of 64 drafts behind long documents, eight query heads per KV head
        {"name": "tree_long", "kind": "tree", "prompts": 8, "samples": 1, "plo": 0, "phi": 0, "olo": 30000,
         "ohi": 131000, "tlo": 64, "thi": 64, "H": 64, "KVH": 8, "D": 128, "page": 64, "lens": 4, "dtype": "bf16"},
        # the drafts of four sequences into their pages, heads normed, the whole head rotated: latency
        {"name": "append_drafts", "kind": "append", "B": 4, "olo": 500, "ohi": 4000, "tlo": 16, "thi": 16, "H": 32,
         "KVH": 8, "D": 128, "R": 128, "layout": "half", "norm": True, "page": 16, "lens": 5, "dtype": "bf16"},
        # prompts of several users: heads normed, half of each head rotated in adjacent pairs
        {"name": "append_prompts_part", "kind": "append", "B": 9, "olo": 300, "ohi": 3001, "tlo": 3001, "thi": 3001,
         "H": 32, "KVH": 8, "D": 128, "R": 64, "layout": "interleaved", "norm": True, "page": 64, "lens": 6,
         "dtype": "bf16"},
        # the positions of a step's 64 drafts, far into a context that the frequencies were scaled for
        {"name": "tables_step", "kind": "tables", "N": 64, "R": 128, "far": 131072, "theta": 500000.0,
         "scaling": "llama3", "layout": "half", "dtype": "bf16"},
        # those of prompts written at once, float32 tables in adjacent pairs
        {"name": "tables_prompts", "kind": "tables", "N": 27001, "R": 128, "far": 1000000, "theta": 10000.0,
         "scaling": "yarn", "layout": "interleaved", "dtype": "f32"},
        # three drafts of one sequence kept in two layers: the smallest call
        {"name": "keep_small", "kind": "keep", "layers": 2, "KVH": 8, "D": 128, "page": 16, "B": 1, "olo": 700,
         "ohi": 700, "T": 8, "most": 3, "lens": 7, "dtype": "bf16"},
        # paths of up to eight of 40 drafts for 64 sequences in 16 layers
        {"name": "keep_wide", "kind": "keep", "layers": 16, "KVH": 8, "D": 128, "page": 16, "B": 64, "olo": 200,
         "ohi": 3000, "T": 40, "most": 8, "lens": 8, "dtype": "bf16"},
        # the next token of four sequences, greedily, under all rules
        {"name": "logits_greedy", "kind": "logits", "B": 4, "olo": 1500, "ohi": 6000, "tlo": 1, "thi": 1, "V": 128256,
         "K": 32, "masked": True, "greedy": True, "lens": 9, "dtype": "f32"},
        # the logits of 16 sequences' trees of 25 drafts, each node with the grammar's mask behind its own path
        {"name": "logits_trees", "kind": "logits", "B": 16, "olo": 1000, "ohi": 20000, "tlo": 25, "thi": 25,
         "V": 128256, "K": 300, "masked": True, "greedy": False, "lens": 10, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "tree", "append", "append", "tables", "keep", "logits", "logits"))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f16")), "lens": rng.randrange(1 << 30)}
    if kind == "tables":
        c.update(N=_log_int(rng, 1, 27000), R=2 * _log_int(rng, 8, 128), far=_log_int(rng, 1000, 1 << 21),
                 theta=rng.choice((10000.0, 500000.0)), scaling=rng.choice(("none", "linear", "ntk", "llama3", "yarn")),
                 layout=rng.choice(("half", "interleaved")), dtype=rng.choice(("bf16", "f16", "f32")))
        return c
    if kind == "logits":
        N = _log_int(rng, 1, 400)
        t = rng.choice((1, 1, _log_int(rng, 1, min(64, N))))
        hi = _log_int(rng, 10, 20000)
        c.update(B=max(1, N // t), olo=_log_int(rng, 5, hi), ohi=hi, tlo=rng.choice((1, t)), thi=t,
                 V=rng.choice((128256, _log_int(rng, 90, 128256))), K=rng.choice((0, _log_int(rng, 1, 500))),
                 masked=rng.random() < 0.6, greedy=rng.random() < 0.5, dtype=rng.choice(("f32", "f32", "bf16", "f16")))
        c["tlo"], c["thi"] = min(c["tlo"], c["olo"]), min(c["thi"], c["olo"])
        return c
    c["page"] = rng.choice((8, 16, 16, 32, 64, 256))
    if kind == "keep":
        T = _log_int(rng, 2, 64)
        lo = _log_int(rng, 20, 1000)
        c.update(layers=rng.randint(1, 16), KVH=rng.choice((1, 4, 8, 8)), D=rng.choice((64, 128, 128)),
                 B=_log_int(rng, 1, 64), olo=lo, ohi=lo + _log_int(rng, 10, 2000), T=T, most=_log_int(rng, 1, T - 1))
        return c
    c["H"], c["KVH"] = rng.choice(HEADS)
    c["D"] = rng.choice((64, 128, 128))
    if kind == "append":
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, max(1, 8000 // B))
        c.update(B=B, olo=hi, ohi=hi + _log_int(rng, 10, 2000), tlo=rng.choice((1, hi)), thi=hi,
                 R=rng.choice((c["D"], c["D"], c["D"] // 2, c["D"] // 4, 8 * rng.randint(1, c["D"] // 8))),
                 layout=rng.choice(("half", "interleaved")), norm=rng.random() < 0.7)
        return c
    prompts, samples = rng.choice(((1, _log_int(rng, 2, 32)), (_log_int(rng, 1, 8), rng.randint(1, 8)),
                                   (_log_int(rng, 1, 32), 1)))
    n = prompts * samples
    t = _log_int(rng, 2, max(3, min(200, 2000 // n)))
    # at most 2^20 cached rows over the KV heads and 2^28 scores
    most = max(t + 1, min((1 << 20) // c["KVH"] // 2, (1 << 27) // (c["H"] * n * t)))
    plo = _log_int(rng, 20, most) if samples > 1 and most > 40 * prompts and rng.random() < 0.9 else 0
    phi = min(int(plo * rng.uniform(1, 3)), most)
    most = max(t + 1, most // n)
    olo = _log_int(rng, t, most)
    c.update(prompts=prompts, samples=samples, plo=plo, phi=max(plo, phi), olo=olo, ohi=rng.randint(olo, most),
             tlo=rng.choice((1, t)), thi=t)
    return c


# ------------------------------------------------------------------- inputs
def _dtype(case):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[case["dtype"]]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(g, pages, page, KVH, D, dtype, keys=False):
    """A page pool [pages, page, KVH, D] ~ N(0, 1); keys get a rank-4 bias per
    KV head besides: scores with the spread of a trained model's."""
    x = torch.randn(pages * page, KVH, D, generator=g, device="cuda")
    if keys:
        C = torch.randn(KVH, pages * page, 4, generator=g, device="cuda")
        U = torch.randn(KVH, 4, D, generator=g, device="cuda") * 0.5
        x += torch.bmm(C, U).permute(1, 0, 2)
    return x.to(dtype).view(pages, page, KVH, D)


def _tree(r, t, spare):
    """Parents of t drafted tokens: the first follows the context, later ones
    mostly early nodes (the wide levels of a draft tree); the last `spare` slots
    are not in use."""
    return [-1] + [int(i * r.random() ** 1.5) for i in range(1, t - spare)] + [-2] * min(spare, t - 1)


def _batch(case):
    """Sequences [(prompt, shared tokens, length, parents of the new tokens)]."""
    r = random.Random(case["lens"])
    seqs = []
    for p in range(case.get("prompts", case.get("B"))):
        P = r.randint(case["plo"], case["phi"]) if "plo" in case else 0
        shared = P // case["page"] * case["page"] if case.get("samples", 1) > 1 else 0
        for _ in range(case.get("samples", 1)):
            n = r.randint(case["olo"], case["ohi"])
            t = min(n, r.randint(case["tlo"], case["thi"]))
            seqs.append((p, shared, P + n, _tree(r, t, r.choice((0, 0, t // 8)))))
    return seqs


def _prefixes(seqs):
    """[(members, shared tokens)] of the prompts that several sequences share."""
    groups = {}
    for i, (p, shared, _, _) in enumerate(seqs):
        if shared:
            groups.setdefault(p, ([], shared))[0].append(i)
    return [g for g in groups.values() if len(g[0]) > 1]


def _table(g, seqs, page):
    """(block table, pages in the pool): pages in random order, the full pages
    of a prompt held once for its samples."""
    prompts = {p: shared // page for p, shared, _, _ in seqs}
    used = [-(-n // page) for _, _, n, _ in seqs]
    total = sum(prompts.values()) + sum(u - prompts[s[0]] for u, s in zip(used, seqs)) + 7
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(seqs), max(used), dtype=torch.int32, device="cuda")
    at, first = 0, {}
    for b, (p, _, _, _) in enumerate(seqs):
        n = prompts[p]
        if p not in first:
            first[p] = at
            at += n
        table[b, :n] = order[first[p]:first[p] + n]
        table[b, n:used[b]] = order[at:at + used[b] - n]
        at += used[b] - n
    return table, total


def _kept(case):
    """(lengths, kept drafts of each sequence): paths whose nodes lie in place or
    behind all the rows that the path moves to, so that a second pass finds what
    the first one found."""
    r = random.Random(case["lens"])
    lens = [r.randint(case["olo"], case["ohi"]) for _ in range(case["B"])]
    kept = []
    for _ in lens:
        n = r.randint(1, case["most"])
        stay = r.randint(0, n - 1)
        kept.append(list(range(stay)) + sorted(r.sample(range(n, case["T"]), min(n - stay, case["T"] - n))))
    return lens, kept


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    st = {"kind": kind, "case": case}
    if kind == "tables":
        st["positions"] = torch.randint(0, case["far"], (case["N"],), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from santa_amd.paged import RopeScaling

            st["scaling"] = None if case["scaling"] == "none" else RopeScaling(case["scaling"], factor=8.0,
                                                                               original_len=8192)
        return st
    if kind == "keep":
        lens, st["kept"] = _kept(case)
        page, T = case["page"], case["T"]
        pages = sum(-(-(n + T) // page) for n in lens) + 2
        if own:
            from santa_amd.paged import PagedKVCache

            st["cache"] = PagedKVCache(case["layers"], pages, page, kv_heads=case["KVH"], head_dim=case["D"],
                                       max_seqs=len(lens), max_len=max(lens) + T, dtype=_dtype(case), device="cuda")
        else:
            st["cache"] = _PlainPages(case["layers"], pages, page, case["KVH"], case["D"], len(lens), max(lens) + T,
                                      _dtype(case))
        for t in (*st["cache"].k, *st["cache"].v):
            t.normal_(generator=g)
        st["seqs"] = st["cache"].add(lens)
        return st
    seqs = _batch(case)
    st["lens"], st["parents"] = [s[2] for s in seqs], [s[3] for s in seqs]
    st["new"] = [len(p) for p in st["parents"]]
    N = sum(st["new"])
    if kind == "logits":
        _prepare_logits(st, g, N)
        H, KVH, prefixes = 1, 1, []
    else:
        H, KVH, D, page, dtype = case["H"], case["KVH"], case["D"], case["page"], _dtype(case)
        prefixes = st["prefixes"] = _prefixes(seqs)
        st["table"], pages = _table(g, seqs, page)
        st["k"] = _pool(g, pages, page, KVH, D, dtype, True)
        st["v"] = _pool(g, pages, page, KVH, D, dtype)
        if kind == "append":
            R = case["R"]
            st["qkv"] = torch.randn(N, H + 2 * KVH, D, generator=g, device="cuda", dtype=dtype)
            angle = torch.rand(N, R // 2, generator=g, device="cuda", dtype=torch.float64) * (2 * math.pi)
            angle = torch.cat([angle, angle], -1) if case["layout"] == "half" else angle.repeat_interleave(2, -1)
            st["cos"], st["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
            st["wq"], st["wk"] = ((torch.rand(D, generator=g, device="cuda") + 0.5).to(dtype) if case["norm"] else None
                                  for _ in range(2))
        else:
            st["q"] = torch.randn(N, H, D, generator=g, device="cuda", dtype=dtype)
    if own:
        from santa_amd.paged import PagedPlan

        st["plan"] = PagedPlan(st["lens"], heads=H, kv_heads=KVH, new_tokens=st["new"], prefixes=prefixes,
                               parents=st["parents"], device="cuda")
    return st


def _prepare_logits(st, g, N):
    case = st["case"]
    V, B = case["V"], len(st["lens"])

    def ids(*size):  # few tokens make up most of a text
        u = torch.rand(*size, generator=g, device="cuda", dtype=torch.float64)
        return (V ** u - 1).long().clamp(0, V - 1)

    st["logits"] = torch.randn(N, V, generator=g, device="cuda").mul_(3.0).to(_dtype(case))
    order = torch.randperm(V, generator=g, device="cuda")
    st["tokens"] = order[ids(B, max(st["lens"]))].to(torch.int32)
    r = random.Random(case["lens"] + 1)
    st["prompts"] = torch.tensor([r.randint(0, n - t) for n, t in zip(st["lens"], st["new"])], dtype=torch.int32).cuda()
    rules = [[r.choice((1.0, r.uniform(1.0, 1.5))) for _ in range(B)], [r.uniform(0.0, 0.5) for _ in range(B)],
             [r.choice((0.0, r.uniform(0.0, 1.0))) for _ in range(B)]]
    st["repetition"], st["frequency"], st["presence"] = (torch.tensor(x, dtype=torch.float32).cuda() for x in rules)
    st["bias"] = st["allowed"] = None
    if case["K"]:
        K = min(case["K"], V)
        at = torch.stack([torch.randperm(V, generator=g, device="cuda")[:K] for _ in range(B)]).to(torch.int32)
        at[:, K // 2 + 1:] = torch.where(torch.arange(B, device="cuda")[:, None] % 3 == 1, -1, at[:, K // 2 + 1:])
        st["bias"] = (at, torch.randn(B, K, generator=g, device="cuda") * 4.0)
    if case["masked"]:
        # from a grammar that leaves a few tokens to one that forbids a few
        share = torch.rand(N, 1, generator=g, device="cuda", dtype=torch.float64) ** 3
        bits = torch.zeros(N, -(-V // 32), dtype=torch.int32, device="cuda")
        for i in range(0, N, 16):
            free = torch.rand(min(16, N - i), 32 * bits.shape[1], generator=g, device="cuda") < share[i:i + 16]
            free[:, 7 % V] = True
            weight = torch.tensor([1 << b if b < 31 else -(1 << 31) for b in range(32)], device="cuda")
            bits[i:i + 16] = (free.view(len(free), -1, 32) * weight).sum(-1).to(torch.int32)
        st["allowed"] = bits


# -------------------------------------------------------------- plain forms
class _PlainPages:
    """Sequences with pages of their own, rows moved by indexing the pools."""

    def __init__(self, layers, pages, page, KVH, D, seqs, widest, dtype):
        self.page = page
        self.k, self.v = ([torch.zeros(pages, page, KVH, D, dtype=dtype, device="cuda") for _ in range(layers)]
                          for _ in range(2))
        self.block_table = torch.zeros(seqs, -(-widest // page), dtype=torch.int32, device="cuda")
        self.free, self.rows, self.lens = list(range(pages)), {}, {}

    def add(self, lengths):
        seqs = list(range(len(lengths)))
        for s in seqs:
            self.rows[s], self.lens[s] = [], 0
        self.extend(seqs, lengths)
        return seqs

    def extend(self, seqs, tokens):
        tokens = [tokens] * len(seqs) if isinstance(tokens, int) else tokens
        edits = []
        for s, t in zip(seqs, tokens):
            self.lens[s] += t
            while len(self.rows[s]) * self.page < self.lens[s]:
                edits.append((s, len(self.rows[s]), self.free[0]))
                self.rows[s].append(self.free.pop(0))
        if edits:
            s, at, page = torch.tensor(edits).t().cuda()
            self.block_table[s, at] = page.to(torch.int32)

    def keep(self, seqs, new_tokens, kept):
        new_tokens = [new_tokens] * len(seqs) if isinstance(new_tokens, int) else new_tokens
        src, dst = [], []
        for s, t, idx in zip(seqs, new_tokens, kept):
            base, row = self.lens[s] - t, self.rows[s]
            for j, i in enumerate(idx):
                if i != j:
                    src.append(row[(base + i) // self.page] * self.page + (base + i) % self.page)
                    dst.append(row[(base + j) // self.page] * self.page + (base + j) % self.page)
            self.lens[s] = base + len(idx)
            used = -(-self.lens[s] // self.page)
            self.free = sorted(self.free + row[used:])
            del row[used:]
        if src:
            src, dst = torch.tensor(src).cuda(), torch.tensor(dst).cuda()
            for t in (*self.k, *self.v):
                t = t.view(-1, *t.shape[2:])
                t[dst] = t[src]


def _run_keep(st):
    """One pass leaves the sequences as long as it found them."""
    cache, seqs, T, kept = st["cache"], st["seqs"], st["case"]["T"], st["kept"]
    cache.extend(seqs, T)
    cache.keep(seqs, T, kept)
    cache.keep(seqs, [len(k) for k in kept], [[] for _ in kept])
    return {"k": list(cache.k), "v": list(cache.v)}


def _frequencies(case):
    """(Angle per position of each pair, in float64; factor of cos and sin)."""
    R, theta, kind = case["R"], case["theta"], case["scaling"]
    i = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    if kind == "ntk":  # the base grows so that the lowest frequency shrinks by the factor
        theta = theta * 8.0 ** (R / (R - 2))
    f = theta ** (-2.0 * i / R)
    if kind == "linear":
        return f / 8.0, 1.0
    turns = 8192 * f / (2 * math.pi)  # over the original length
    if kind == "llama3":  # below 1 turn scaled, above 4 left
        keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        return f / 8.0 * (1 - keep) + f * keep, 1.0
    if kind == "yarn":  # scaled from the pair of 1 turn on, left up to the pair of 32
        at = [R * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / 8.0 * ramp + f * (1 - ramp), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _plain_tables(st):
    case = st["case"]
    f, up = _frequencies(case)
    angle = st["positions"].double()[:, None] * f
    cos, sin = angle.cos() * up, angle.sin() * up
    if case["layout"] == "half":
        cos, sin = torch.cat([cos, cos], -1), torch.cat([sin, sin], -1)
    else:
        cos, sin = cos.repeat_interleave(2, -1), sin.repeat_interleave(2, -1)
    return {"cos": cos.to(_dtype(case)), "sin": sin.to(_dtype(case))}


def _slots(st):
    """(Token of the batch, sequence, position) of the new tokens in use."""
    token, seq, pos, t0 = [], [], [], 0
    for b, (n, parents) in enumerate(zip(st["lens"], st["parents"])):
        for i, p in enumerate(parents):
            if p > -2:
                token.append(t0 + i)
                seq.append(b)
                pos.append(n - len(parents) + i)
        t0 += len(parents)
    return (torch.tensor(x, device="cuda") for x in (token, seq, pos))


def _plain_append(st):
    case = st["case"]
    H, KVH, D, R, page = case["H"], case["KVH"], case["D"], case["R"], case["page"]
    x = st["qkv"][:, :H + KVH].float()
    if case["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        x = torch.cat([x[:, :H] * st["wq"].float(), x[:, H:] * st["wk"].float()], 1)
    y, c, s = x[..., :R], st["cos"].float()[:, None], st["sin"].float()[:, None]
    if case["layout"] == "half":
        other = torch.cat([-y[..., R // 2:], y[..., :R // 2]], -1)
    else:
        other = torch.stack([-y[..., 1::2], y[..., ::2]], -1).flatten(-2)
    turned = torch.cat([y * c + other * s, x[..., R:]], -1).to(st["qkv"].dtype)
    token, seq, pos = _slots(st)
    at = st["table"][seq, pos // page].long() * page + pos % page
    st["k"].view(-1, KVH, D)[at] = turned[token, H:]
    st["v"].view(-1, KVH, D)[at] = st["qkv"][token, H + KVH:]
    return {"q": turned[:, :H], "k": st["k"], "v": st["v"]}


def _sees(parents):
    """[t, t]: the drafted tokens that each one follows, itself among them."""
    t = len(parents)
    sees = [[False] * t for _ in range(t)]
    for i, p in enumerate(parents):
        if p > -2:
            if p >= 0:
                sees[i] = list(sees[p])
            sees[i][i] = True
    return torch.tensor(sees)


def _plain_tree(st):
    case = st["case"]
    H, KVH, D, page = case["H"], case["KVH"], case["D"], case["page"]
    G, scale = H // KVH, 1.0 / math.sqrt(D)
    out, t0 = torch.empty_like(st["q"]), 0
    for b, (n, parents) in enumerate(zip(st["lens"], st["parents"])):
        t = len(parents)
        at = torch.arange(n, device="cuda")
        at = st["table"][b, at // page].long() * page + at % page
        k, v = (x.view(-1, KVH, D)[at].float().permute(1, 0, 2).contiguous() for x in (st["k"], st["v"]))
        q = st["q"][t0:t0 + t].float().view(t, KVH, G, D).permute(1, 0, 2, 3).reshape(KVH, t * G, D)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(KVH, t, G, n) * scale
        s[..., n - t:].masked_fill_(~_sees(parents).cuda()[None, :, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.bmm(p.view(KVH, t * G, n), v) / p.view(KVH, t * G, n).sum(-1, keepdim=True)
        o = o.view(KVH, t, G, D).permute(1, 0, 2, 3).reshape(t, H, D)
        used = torch.tensor([x > -2 for x in parents], device="cuda")
        out[t0:t0 + t] = torch.where(used[:, None, None], o, 0.0).to(out.dtype)
        t0 += t
    return {"out": out}


def _plain_logits(st):
    case = st["case"]
    V, N = case["V"], len(st["logits"])
    out = torch.empty(N, V, device="cuda")
    at, i = torch.arange(V, device="cuda"), 0
    for b, (n, parents) in enumerate(zip(st["lens"], st["parents"])):
        t = len(parents)
        row, place = st["tokens"][b, :n].long(), torch.arange(n - t, device="cuda")
        used = torch.tensor([[p > -2] for p in parents], device="cuda").long()
        said, told = (torch.zeros(V, dtype=torch.long, device="cuda").index_add_(0, row[:n - t], x.long())
                      for x in (place >= st["prompts"][b], place < st["prompts"][b]))
        count = (said * used).index_add_(1, row[n - t:], _sees(parents).cuda().long())
        seen = count + told * used > 0
        x, r = st["logits"][i:i + t].float(), st["repetition"][b]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x) - st["frequency"][b] * count.float()
        x = torch.where(count > 0, x - st["presence"][b], x)
        if st["bias"] is not None:
            ids, values = (y[b] for y in st["bias"])
            x[:, ids[ids >= 0].long()] += values[ids >= 0]
        if st["allowed"] is not None:
            x = torch.where((st["allowed"][i:i + t, at >> 5] >> (at & 31)) & 1 > 0, x, -math.inf)
        out[i:i + t] = x
        i += t
    return {"token": out.argmax(-1)} if case["greedy"] else {"logits": out}


def run(state):
    kind, case = state["kind"], state["case"]
    if kind == "keep":
        return _run_keep(state)
    if not own:
        return {"tree": _plain_tree, "append": _plain_append, "tables": _plain_tables, "logits": _plain_logits}[kind](state)
    if kind == "tree":
        from santa_amd.paged import paged_attention

        return {"out": paged_attention(state["q"], state["k"], state["v"], state["table"], state["plan"])}
    if kind == "append":
        from santa_amd.paged import rope_append

        q = rope_append(state["qkv"], state["cos"], state["sin"], state["k"], state["v"], state["table"], state["plan"],
                        q_norm=state["wq"], k_norm=state["wk"], eps=EPS, interleaved=case["layout"] == "interleaved")
        return {"q": q, "k": state["k"], "v": state["v"]}
    if kind == "tables":
        from santa_amd.paged import rope_tables

        cos, sin = rope_tables(state["positions"], case["R"], theta=case["theta"], scaling=state["scaling"],
                               interleaved=case["layout"] == "interleaved", dtype=_dtype(case))
        return {"cos": cos, "sin": sin}
    from santa_amd.logits import adjust_logits

    out = adjust_logits(state["logits"], state["tokens"], state["plan"], prompts=state["prompts"],
                        repetition=state["repetition"], frequency=state["frequency"], presence=state["presence"],
                        bias=state["bias"], allowed=state["allowed"], greedy=case["greedy"])
    return {"token" if case["greedy"] else "logits": out}


# --------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "tables":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 4.0 * case["N"] + 2.0 * size * case["N"] * case["R"], "flops": 2.0 * case["N"] * case["R"]}
    if kind == "keep":
        moved = sum(i != j for idx in _kept(case)[1] for j, i in enumerate(idx))
        return {"bytes": 2.0 * moved * case["layers"] * 2 * case["KVH"] * case["D"] * 2, "flops": 0.0}
    seqs = _batch(case)
    N = sum(len(s[3]) for s in seqs)
    if kind == "logits":
        V, size = case["V"], 4 if case["dtype"] == "f32" else 2
        read = N * V * size + 4 * sum(s[2] for s in seqs) + 8 * len(seqs) * min(case["K"], V)
        return {"bytes": float(read + (N * -(-V // 32) * 4 if case["masked"] else 0) + N * (8 if case["greedy"] else 4 * V)),
                "flops": 4.0 * N * V}
    H, KVH, D = case["H"], case["KVH"], case["D"]
    if kind == "append":
        return {"bytes": 2.0 * N * (2 * (H + 2 * KVH) * D + 2 * case["R"]),
                "flops": (3.0 * case["R"] + (4.0 * D if case["norm"] else 0.0)) * N * (H + KVH)}
    prefix = {b: P for members, P in _prefixes(seqs) for b in members}
    tokens = sum(P for _, P in _prefixes(seqs)) + sum(s[2] - prefix.get(b, 0) for b, s in enumerate(seqs))
    pairs = 0.0
    for _, _, n, parents in seqs:
        depth = []
        for p in parents:
            depth.append(0 if p == -2 else 1 + (depth[p] if p >= 0 else 0))
        pairs += sum(n - len(parents) + d for d in depth if d)
    return {"bytes": 4.0 * tokens * KVH * D + 4.0 * N * H * D, "flops": 4.0 * pairs * H * D}


# -------------------------------------------------------------------- exact
def _exact_tree(st):
    """Token by token of a sequence the keys on its path, head by head, in float64."""
    case = st["case"]
    H, KVH, D, page = case["H"], case["KVH"], case["D"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, parents) in enumerate(zip(st["lens"], st["parents"])):
        t = len(parents)
        hidden = torch.zeros(t, n, dtype=torch.bool)
        for i, p in enumerate(parents):
            hidden[i, n - t:] = True
            at = i if p > -2 else -1
            while at >= 0:  # up to the root
                hidden[i, n - t + at] = False
                at = parents[at]
        hidden = hidden.cuda()
        used = [i for i, p in enumerate(parents) if p > -2]
        where = torch.tensor([int(x) * page for x in st["table"][b, :-(-n // page)].tolist()], device="cuda")
        where = (where[:, None] + torch.arange(page, device="cuda")).flatten()[:n]
        for kv in range(KVH):
            k = st["k"].view(-1, KVH, D)[where, kv].double().t().contiguous()
            v = st["v"].view(-1, KVH, D)[where, kv].double()
            for h in range(kv * (H // KVH), (kv + 1) * (H // KVH)):
                s = (st["q"][start:start + t, h].double() @ k) / math.sqrt(D)
                o = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
                out[[start + i for i in used], h] = o[used]
        start += t
    return {"out": out}


def _exact_append(st):
    case = st["case"]
    H, KVH, D, R, page = case["H"], case["KVH"], case["D"], case["R"], case["page"]
    x = st["qkv"].double()
    if case["norm"]:
        size = (x * x).sum(-1, keepdim=True) / D
        w = torch.ones(H + 2 * KVH, D, dtype=torch.float64, device="cuda")
        w[:H], w[H:H + KVH] = st["wq"].double(), st["wk"].double()
        normed = x / torch.sqrt(size + EPS) * w
        x = torch.cat([normed[:, :H + KVH], x[:, H + KVH:]], 1)
    first = torch.arange(R // 2, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (R // 2 if case["layout"] == "half" else 1)
    c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]
    turned = x.clone()
    turned[:, :H + KVH, first] = (x[..., first] * c[..., first] - x[..., second] * s[..., first])[:, :H + KVH]
    turned[:, :H + KVH, second] = (x[..., second] * c[..., second] + x[..., first] * s[..., second])[:, :H + KVH]
    k, v = st["k"].double(), st["v"].double()
    table, tokens, where, t0 = st["table"].tolist(), [], [], 0
    for row, n, parents in zip(table, st["lens"], st["parents"]):
        used = [i for i, p in enumerate(parents) if p > -2]
        tokens += [t0 + i for i in used]
        where += [row[p // page] * page + p % page for p in (n - len(parents) + i for i in used)]
        t0 += len(parents)
    where, tokens = torch.tensor(where, device="cuda"), torch.tensor(tokens, device="cuda")
    k.view(-1, KVH, D).index_copy_(0, where, turned[tokens, H:H + KVH].contiguous())
    v.view(-1, KVH, D).index_copy_(0, where, x[tokens, H + KVH:].contiguous())
    return {"q": turned[:, :H], "k": k, "v": v}


def _exact_tables(st):
    """Pair by pair from the published rules, positions reduced to one turn."""
    case = st["case"]
    R, theta, kind = case["R"], case["theta"], case["scaling"]
    pos = st["positions"].double()
    cos, sin = (torch.empty(len(pos), R, dtype=torch.float64, device="cuda") for _ in range(2))
    up = 1.0 + 0.1 * math.log(8.0) if kind == "yarn" else 1.0
    if kind == "ntk":
        theta *= 8.0 ** (R / (R - 2.0))
    for i in range(R // 2):
        f = theta ** (-2.0 * i / R)
        length = 2 * math.pi / f
        if kind == "linear":
            f /= 8.0
        elif kind == "llama3":
            if length > 8192 / 1.0:
                f /= 8.0
            elif length > 8192 / 4.0:
                smooth = (8192 / length - 1.0) / (4.0 - 1.0)
                f = (1.0 - smooth) * f / 8.0 + smooth * f
        elif kind == "yarn":
            lo, hi = (R * math.log(8192 / (beta * 2 * math.pi)) / (2 * math.log(theta)) for beta in (32, 1))
            lo, hi = max(0, math.floor(lo)), min(R - 1, math.ceil(hi))
            share = min(1.0, max(0.0, (i - lo) / (hi - lo if hi > lo else 0.001)))
            f = f * (1.0 - share) + f / 8.0 * share
        turn = torch.remainder(pos * f, 2 * math.pi)
        for j in ((i, i + R // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)):
            cos[:, j], sin[:, j] = up * torch.cos(turn), up * torch.sin(turn)
    return {"cos": cos, "sin": sin}


def _exact_logits(st):
    case = st["case"]
    V, N = case["V"], len(st["logits"])
    out = torch.empty(N, V, dtype=torch.float64, device="cuda")
    i = 0
    for b, (n, parents) in enumerate(zip(st["lens"], st["parents"])):
        t, prompt = len(parents), int(st["prompts"][b])
        row = st["tokens"][b].long()
        r, f, p = (float(st[name][b]) for name in ("repetition", "frequency", "presence"))
        told = torch.bincount(row[:min(prompt, n - t)], minlength=V)
        said = torch.bincount(row[min(prompt, n - t):n - t], minlength=V)
        for j, parent in enumerate(parents):
            count, seen = (said.clone(), told + said > 0) if parent > -2 else (torch.zeros_like(said), told < 0)
            at = j if parent > -2 else -1
            while at >= 0:
                count[row[n - t + at]] += 1
                seen[row[n - t + at]] = True
                at = parents[at]
            x = st["logits"][i].double()
            x[seen] = torch.where(x[seen] > 0, x[seen] / r, x[seen] * r)
            x = x - f * count.double() - p * (count > 0).double()
            if st["bias"] is not None:
                for_row = st["bias"][0][b] >= 0
                x[st["bias"][0][b][for_row].long()] += st["bias"][1][b][for_row].double()
            if st["allowed"] is not None:
                shifts = torch.arange(32, device="cuda", dtype=torch.int32)
                free = (st["allowed"][i][:, None] >> shifts & 1).flatten()[:V].bool()
                x[~free] = -math.inf
            out[i] = x
            i += 1
    return {"token": out.argmax(-1)} if case["greedy"] else {"logits": out}


def _exact_keep(case, seed):
    """Row by row, from copies of the pools."""
    st = prepare(case, seed)
    lens, kept = _kept(case)
    page, T, table = case["page"], case["T"], []
    at = 0
    for n in lens:  # pages are taken lowest number first: the contexts', then the drafts'
        table.append(list(range(at, at + -(-n // page))))
        at += -(-n // page)
    for n, row in zip(lens, table):
        more = -(-(n + T) // page) - len(row)
        row += range(at, at + more)
        at += more
    res = {}
    for name in ("k", "v"):
        res[name] = []
        for t in getattr(st["cache"], name):
            new = t.clone()
            for n, row, idx in zip(lens, table, kept):
                for j, i in enumerate(idx):
                    new[row[(n + j) // page], (n + j) % page] = t[row[(n + i) // page], (n + i) % page]
            res[name].append(new)
    return res


def exact(case, seed):
    if case["kind"] == "keep":
        return _exact_keep(case, seed)
    st = prepare(case, seed)
    return {"tree": _exact_tree, "append": _exact_append, "tables": _exact_tables, "logits": _exact_logits}[case["kind"]](st)
