"""The operators of a shared paged cache and what they are timed on: forking,
copying, freeing and compacting pages (``PagedKVCache``), the exact attention
over pages for batches that share prompt prefixes, with one or several new
tokens per sequence (``paged_attention``), and RoPE with the write of new
tokens into their pages (``rope_append``).

Shapes are the repository's own (32q/8kv, 64q/8kv, 28q/4kv and 32q/32kv heads,
head_dim 128 or 64, 16-token pages and larger ones, prompts up to 131072 tokens,
layers of the Llama-3.1-8B dimensions) or generic.
"""
import math
import random

import torch

own = False

HEADS = ((32, 8), (32, 8), (64, 8), (28, 4), (32, 32), (16, 8), (12, 1))


def listed():
    return [
        # two more answers asked for a short chat turn, two layers: the smallest call, latency bound
        {"name": "fork_short", "kind": "fork", "layers": 2, "KVH": 8, "D": 128, "page": 16, "others": "700 300",
         "len": 1500, "n": 2, "dtype": "bf16"},
        # 64 samples of one long prompt: their table rows, and the partly filled last page copied for each
        {"name": "fork_wide", "kind": "fork", "layers": 16, "KVH": 8, "D": 128, "page": 16, "others": "5000",
         "len": 32760, "n": 64, "dtype": "bf16"},
        # half of a batch has finished and its pages are closed up, 32-token pages
        {"name": "compact_half", "kind": "compact", "layers": 8, "KVH": 8, "D": 128, "page": 32, "others": "9000",
         "lo": 500, "hi": 6000, "seqs": 16, "lens": 5, "dtype": "f16"},
        # four samples of a short prompt: the smallest attention call, launch and latency bound
        {"name": "attend_small", "kind": "attend", "prompts": 1, "samples": 4, "plo": 1000, "phi": 1000, "olo": 60,
         "ohi": 100, "tlo": 1, "thi": 1, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 1, "mixed": False,
         "dtype": "bf16"},
        # 64 sequences behind one 32k-token prompt, each some way into its answer
        {"name": "attend_shared_32k", "kind": "attend", "prompts": 1, "samples": 64, "plo": 32768, "phi": 32768,
         "olo": 100, "ohi": 2000, "tlo": 1, "thi": 1, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 2,
         "mixed": False, "dtype": "bf16"},
        # the largest: 32 sequences behind a 128k-token document, eight query heads per KV head
        {"name": "attend_shared_128k", "kind": "attend", "prompts": 1, "samples": 32, "plo": 131001, "phi": 131001,
         "olo": 200, "ohi": 4000, "tlo": 1, "thi": 1, "H": 64, "KVH": 8, "D": 128, "page": 64, "lens": 3,
         "mixed": False, "dtype": "bf16"},
        # several prompts with some samples each, arrived in any order, odd lengths, seven heads per KV head
        {"name": "attend_prompts_f16", "kind": "attend", "prompts": 5, "samples": 6, "plo": 900, "phi": 9001,
         "olo": 1, "ohi": 1500, "tlo": 1, "thi": 1, "H": 28, "KVH": 4, "D": 128, "page": 32, "lens": 4, "mixed": True,
         "dtype": "f16"},
        # continuous batching without anything shared: exact decode over pages
        {"name": "attend_unshared", "kind": "attend", "prompts": 16, "samples": 1, "plo": 0, "phi": 0, "olo": 1000,
         "ohi": 40000, "tlo": 1, "thi": 1, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 16, "mixed": False,
         "dtype": "bf16"},
        # drafted tokens verified, five per sequence, head_dim 64
        {"name": "attend_drafts", "kind": "attend", "prompts": 8, "samples": 1, "plo": 0, "phi": 0, "olo": 3000,
         "ohi": 16000, "tlo": 5, "thi": 5, "H": 32, "KVH": 8, "D": 64, "page": 16, "lens": 6, "mixed": False,
         "dtype": "bf16"},
        # users' own prompts behind a system prompt: prefill of the new tokens only
        {"name": "attend_extend", "kind": "attend", "prompts": 1, "samples": 6, "plo": 4000, "phi": 4000, "olo": 100,
         "ohi": 1300, "tlo": 1300, "thi": 1300, "H": 32, "KVH": 8, "D": 128, "page": 16, "lens": 7, "mixed": False,
         "dtype": "bf16"},
        # the new token of each of 64 sequences into its page
        {"name": "append_step", "kind": "append", "B": 64, "olo": 500, "ohi": 4000, "tlo": 1, "thi": 1, "H": 32,
         "KVH": 8, "D": 128, "page": 16, "lens": 8, "dtype": "bf16"},
        # prompts of several users written at once
        {"name": "append_prompts", "kind": "append", "B": 9, "olo": 300, "ohi": 3001, "tlo": 3001, "thi": 3001, "H": 32,
         "KVH": 8, "D": 128, "page": 64, "lens": 9, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("fork", "compact", "attend", "attend", "attend", "attend", "append"))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f16")), "lens": rng.randrange(1 << 30)}
    c["page"] = rng.choice((8, 16, 16, 32, 64, 256))
    if kind in ("fork", "compact"):
        c.update(layers=rng.randint(1, 8), KVH=rng.choice((1, 4, 8, 8)), D=rng.choice((64, 128, 128)))
        c["others"] = " ".join(str(_log_int(rng, 50, 4000)) for _ in range(rng.randint(0, 3)))
        if kind == "fork":
            c.update(len=_log_int(rng, 1, 20000), n=_log_int(rng, 1, min(64, 2048 // c["page"])))
        else:
            lo = _log_int(rng, 30, 1000)
            c.update(lo=lo, hi=lo + _log_int(rng, 10, 2000), seqs=rng.randint(2, 16))
        return c
    c["H"], c["KVH"] = rng.choice(HEADS)
    c["D"] = rng.choice((64, 128, 128))
    if kind == "append":
        B = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, max(1, 8000 // B))
        c.update(B=B, olo=hi, ohi=hi + _log_int(rng, 10, 2000), tlo=1, thi=hi)
        return c
    prompts, samples = rng.choice(((1, _log_int(rng, 2, 64)), (_log_int(rng, 1, 8), rng.randint(1, 12)),
                                   (_log_int(rng, 1, 32), 1)))
    n = prompts * samples
    t = rng.choice((1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, max(17, 2000 // n))))
    # at most 2^20 cached rows over the KV heads and 2^28 scores
    most = max(2, min((1 << 20) // c["KVH"] // 2, (1 << 27) // (c["H"] * n * t)))
    shared = samples > 1 and rng.random() < 0.9
    plo = _log_int(rng, min(20, most // prompts), most // prompts) if shared and most > 2 * prompts else 0
    phi = min(int(plo * rng.uniform(1, 3)), most // prompts)
    most = max(2, most // n) if t == 1 else max(2, min(most, (1 << 20) // c["KVH"] // (2 * n)))
    olo = _log_int(rng, 1, most)
    c.update(prompts=prompts, samples=samples, plo=plo, phi=max(plo, phi), olo=olo, ohi=rng.randint(olo, most),
             tlo=rng.choice((1, t)), thi=t, mixed=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


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


def _batch(case):
    """Sequences [(prompt, shared tokens, length, new tokens)] in the order in
    which the batch holds them."""
    r = random.Random(case["lens"])
    seqs = []
    for p in range(case.get("prompts", case.get("B"))):
        P = r.randint(case["plo"], case["phi"]) if "plo" in case else 0
        shared = P // case["page"] * case["page"] if case.get("samples", 1) > 1 else 0
        for _ in range(case.get("samples", 1)):
            n = r.randint(case["olo"], case["ohi"])
            seqs.append((p, shared, P + n, min(n, r.randint(case["tlo"], case["thi"]))))
    if case.get("mixed"):
        r.shuffle(seqs)
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


def _pages_state(case):
    """(pages, widest row, lengths of the sequences that stay, lengths of the
    pass): what a cache for this case has to hold."""
    page, others = case["page"], [int(n) for n in case["others"].split()]
    if case["kind"] == "fork":
        stay, come = others + [case["len"]], [case["len"] + 1] * case["n"]
        pages = sum(-(-n // page) for n in stay) + 2 * case["n"]
    else:
        r = random.Random(case["lens"])
        stay, come = others, [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
        pages = sum(-(-n // page) for n in stay + come)
    return pages + 3, max(stay + come), stay, come


def prepare(case, seed):
    kind, dtype, page, KVH, D = case["kind"], _dtype(case), case["page"], case["KVH"], case["D"]
    g = _gen(seed)
    st = {"kind": kind, "case": case}
    if kind in ("fork", "compact"):
        pages, widest, stay, come = _pages_state(case)
        seqs = len(stay) + len(come)
        if own:
            from santa_amd.paged import PagedKVCache

            st["cache"] = PagedKVCache(case["layers"], pages, page, kv_heads=KVH, head_dim=D, max_seqs=seqs,
                                       max_len=widest, dtype=dtype, device="cuda")
        else:
            st["cache"] = _PlainPages(case["layers"], pages, page, KVH, D, seqs, widest, dtype)
        for t in st["cache"].k + st["cache"].v:
            t.normal_(generator=g)
        st["stay"] = st["cache"].add(stay)
        st["come"] = come
        return st
    seqs = _batch(case)
    st["lens"], st["new"] = [s[2] for s in seqs], [s[3] for s in seqs]
    st["prefixes"] = _prefixes(seqs)
    st["table"], pages = _table(g, seqs, page)
    st["k"], st["v"] = _pool(g, pages, page, KVH, D, dtype, True), _pool(g, pages, page, KVH, D, dtype)
    N, H = sum(st["new"]), case["H"]
    if kind == "append":
        st["qkv"] = torch.randn(N, H + 2 * KVH, D, generator=g, device="cuda", dtype=dtype)
        angle = torch.rand(N, D // 2, generator=g, device="cuda", dtype=torch.float64) * (2 * math.pi)
        angle = torch.cat([angle, angle], -1)
        st["cos"], st["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    else:
        st["q"] = torch.randn(N, H, D, generator=g, device="cuda", dtype=dtype)
    if own:
        from santa_amd.paged import PagedPlan

        st["plan"] = PagedPlan(st["lens"], heads=H, kv_heads=KVH, new_tokens=st["new"], prefixes=st["prefixes"],
                               device="cuda")
    return st


# -------------------------------------------------------------- plain forms
class _PlainPages:
    """Page bookkeeping on host tensors, page copies as indexing of the pools."""

    def __init__(self, layers, pages, page, KVH, D, seqs, widest, dtype):
        self.page = page
        self.k, self.v = ([torch.zeros(pages, page, KVH, D, dtype=dtype, device="cuda") for _ in range(layers)]
                          for _ in range(2))
        self.block_table = torch.zeros(seqs, -(-widest // page), dtype=torch.int32, device="cuda")
        self.host = torch.zeros(self.block_table.shape, dtype=torch.int64)
        self.refs = torch.zeros(pages, dtype=torch.int64)
        self.lens = {}

    def _used(self, s):
        return -(-self.lens[s] // self.page)

    def _upload(self, rows):
        rows = torch.tensor(rows, dtype=torch.int64)
        self.block_table[rows.cuda()] = self.host[rows].to(torch.int32).cuda()

    def _copy(self, src, dst):
        if len(src):
            src, dst = src.cuda(), dst.cuda()
            for t in self.k + self.v:
                t[dst] = t[src]

    def add(self, lengths):
        seqs = [s for s in range(len(self.host)) if s not in self.lens][:len(lengths)]
        self.lens.update((s, 0) for s in seqs)
        self.extend(seqs, lengths)
        return seqs

    def fork(self, seq, n):
        kids = [s for s in range(len(self.host)) if s not in self.lens][:n]
        used = self._used(seq)
        for s in kids:
            self.lens[s] = self.lens[seq]
            self.host[s, :used] = self.host[seq, :used]
        self.refs[self.host[seq, :used]] += n
        self._upload(kids)
        return kids

    def extend(self, seqs, tokens):
        tokens = [tokens] * len(seqs) if isinstance(tokens, int) else tokens
        free = (self.refs == 0).nonzero()[:, 0]
        at, src, dst = 0, [], []
        for s, t in zip(seqs, tokens):
            used = self._used(s)
            if t and self.lens[s] % self.page:
                last = int(self.host[s, used - 1])
                if self.refs[last] > 1:
                    self.refs[last] -= 1
                    src.append(last)
                    dst.append(int(free[at]))
                    self.host[s, used - 1] = free[at]
                    at += 1
            self.lens[s] += t
            more = self._used(s) - used
            self.host[s, used:used + more] = free[at:at + more]
            at += more
        self.refs[free[:at]] = 1
        self._copy(torch.tensor(src, dtype=torch.int64), torch.tensor(dst, dtype=torch.int64))
        self._upload(seqs)

    def free(self, seqs):
        for s in seqs:
            self.refs[self.host[s, :self._used(s)]] -= 1
            del self.lens[s]

    def compact(self):
        live = (self.refs > 0).nonzero()[:, 0]
        n = len(live)
        src, dst = live[live >= n], (self.refs[:n] == 0).nonzero()[:, 0]
        to = torch.arange(len(self.refs))
        to[src] = dst
        self.refs[dst], self.refs[src] = self.refs[src], 0
        self._copy(src, dst)
        for s in self.lens:
            self.host[s, :self._used(s)] = to[self.host[s, :self._used(s)]]
        self._upload(sorted(self.lens))


def _run_pages(st):
    """One pass leaves the cache's bookkeeping as it found it: the forks or
    the batch that came are gone again at its end."""
    cache, case, page = st["cache"], st["case"], st["case"]["page"]
    if st["kind"] == "fork":
        parent = st["stay"][-1]
        kids = cache.fork(parent, case["n"])
        cache.extend(kids, 1)
        table = [cache.block_table[kids[0]:kids[0] + case["n"], :case["len"] // page + 1]]
        cache.free(kids)
    else:
        came = cache.add(st["come"])
        cache.free(came[::2])
        cache.compact()
        table = [cache.block_table[s, :-(-n // page)] for s, n in zip(came[1::2], st["come"][1::2])]
        cache.free(came[1::2])
    return {"k": cache.k, "v": cache.v, "table": table}


def _rows(st):
    """(sequence, position) of every new token."""
    seq, pos = [], []
    for b, (n, t) in enumerate(zip(st["lens"], st["new"])):
        seq += [b] * t
        pos += range(n - t, n)
    return torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda")


def _tokens(st, b, lo, hi):
    """Pool rows of positions lo .. hi - 1 of sequence b."""
    page = st["case"]["page"]
    at = torch.arange(lo, hi, device="cuda")
    return st["table"][b, at // page].long() * page + at % page


def _part(q, k, v, limit, scale):
    """Maximum, mass and weighted sum of q [KVH, R, D] over k, v [KVH, n, D];
    row r sees the first limit[r] of them (all, where limit is None)."""
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    if limit is not None:
        s = torch.where(torch.arange(k.shape[1], device="cuda")[None, None] < limit[None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    return m, p.sum(-1, keepdim=True), torch.bmm(p, v)


def _plain_attend(st):
    case = st["case"]
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G, scale = H // KVH, 1.0 / math.sqrt(D)
    kf, vf = st["k"].view(-1, KVH, D), st["v"].view(-1, KVH, D)
    starts = [0]
    for t in st["new"]:
        starts.append(starts[-1] + t)

    def keys(b, lo, hi):
        at = _tokens(st, b, lo, hi)
        return (t[at].float().permute(1, 0, 2).contiguous() for t in (kf, vf))

    def rows(at):  # [tokens, H, D] -> [KVH, tokens * G, D]
        return st["q"][at].float().view(-1, KVH, G, D).permute(1, 0, 2, 3).reshape(KVH, -1, D)

    shared, first = {}, {}
    for members, P in st["prefixes"]:
        k, v = keys(members[0], 0, P)
        at = torch.cat([torch.arange(starts[b], starts[b + 1]) for b in members]).cuda()
        q, step = rows(at), max(1, (1 << 28) // (KVH * P))
        parts = [_part(q[:, i:i + step], k, v, None, scale) for i in range(0, q.shape[1], step)]
        m, l, o = (torch.cat(x, 1) for x in zip(*parts))
        i = 0
        for b in members:
            n = st["new"][b] * G
            shared[b], first[b] = tuple(x[:, i:i + n] for x in (m, l, o)), P
            i += n
    out = torch.empty(starts[-1], H, D, dtype=st["q"].dtype, device="cuda")
    for b, (n, t) in enumerate(zip(st["lens"], st["new"])):
        lo = first.get(b, 0)
        limit = torch.arange(n - t - lo + 1, n - lo + 1, device="cuda").repeat_interleave(G)
        m, l, o = _part(rows(slice(starts[b], starts[b + 1])), *keys(b, lo, n), limit, scale)
        if b in shared:
            m2, l2, o2 = shared[b]
            top = torch.maximum(m, m2)
            w, w2 = torch.exp(m - top), torch.exp(m2 - top)
            l, o = l * w + l2 * w2, o * w + o2 * w2
        o = (o / l).view(KVH, t, G, D).permute(1, 0, 2, 3).reshape(t, H, D)
        out[starts[b]:starts[b + 1]] = o.to(out.dtype)
    return {"out": out}


def _plain_append(st):
    case = st["case"]
    H, KVH, D, page = case["H"], case["KVH"], case["D"], case["page"]
    x = st["qkv"].float()
    cos, sin = st["cos"].float()[:, None], st["sin"].float()[:, None]
    half = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    turned = (x * cos + half * sin)[:, :H + KVH].to(st["qkv"].dtype)
    seq, pos = _rows(st)
    at = st["table"][seq, pos // page].long() * page + pos % page
    st["k"].view(-1, KVH, D)[at] = turned[:, H:]
    st["v"].view(-1, KVH, D)[at] = st["qkv"][:, H + KVH:]
    return {"q": turned[:, :H], "k": st["k"], "v": st["v"]}


def run(state):
    kind = state["kind"]
    if kind in ("fork", "compact"):
        return _run_pages(state)
    if not own:
        return _plain_attend(state) if kind == "attend" else _plain_append(state)
    if kind == "attend":
        from santa_amd.paged import paged_attention

        return {"out": paged_attention(state["q"], state["k"], state["v"], state["table"], state["plan"])}
    from santa_amd.paged import rope_append

    q = rope_append(state["qkv"], state["cos"], state["sin"], state["k"], state["v"], state["table"], state["plan"])
    return {"q": q, "k": state["k"], "v": state["v"]}


# --------------------------------------------------------------------- work
def work(case):
    kind, KVH, D, page = case["kind"], case["KVH"], case["D"], case["page"]
    if kind in ("fork", "compact"):
        pages, _, stay, come = _pages_state(case)
        if kind == "fork":
            moved = case["n"] if case["len"] % page else 0
            entries = sum(-(-n // page) for n in come)
        else:
            used = [-(-n // page) for n in come]
            base = sum(-(-n // page) for n in stay)
            live = base + sum(used[1::2])
            at, moved = base, 0
            for i, u in enumerate(used):  # pages of the odd ones beyond the live count move
                moved += max(0, min(u, at + u - live)) if i % 2 else 0
                at += u
            entries = sum(used)
        return {"bytes": 2.0 * moved * case["layers"] * 2 * page * KVH * D * 2 + 4.0 * entries, "flops": 0.0}
    seqs, H = _batch(case), case["H"]
    N = sum(t for _, _, _, t in seqs)
    if kind == "append":
        return {"bytes": 2.0 * N * (2 * (H + 2 * KVH) * D + 2 * D), "flops": 4.0 * N * (H + KVH) * D}
    prefix = {b: P for members, P in _prefixes(seqs) for b in members}
    tokens = sum(P for _, P in _prefixes(seqs)) + sum(n - prefix.get(b, 0) for b, (_, _, n, _) in enumerate(seqs))
    pairs = sum(t * n - t * (t - 1) / 2.0 for _, _, n, t in seqs)
    return {"bytes": 4.0 * tokens * KVH * D + 4.0 * N * H * D, "flops": 4.0 * pairs * H * D}


# -------------------------------------------------------------------- exact
def _exact_pages(case, seed):
    """The pools and table rows after the pass, page by page."""
    st = prepare(case, seed)
    cache, page = st["cache"], case["page"]
    pages, _, stay, come = _pages_state(case)
    base, held = 0, []
    for n in stay:
        held.append(list(range(base, base + -(-n // page))))
        base += -(-n // page)
    moves, rows = [], []
    if case["kind"] == "fork":
        for i in range(case["n"]):
            row = held[-1] + [base + i]
            if case["len"] % page:
                moves.append((held[-1][-1], base + i))
                row = held[-1][:-1] + [base + i]
            rows.append(row)
    else:
        at = base
        for n in come:
            rows.append(list(range(at, at + -(-n // page))))
            at += -(-n // page)
        holes = sorted(p for r in rows[::2] for p in r)
        rows = rows[1::2]
        live = base + sum(len(r) for r in rows)
        high = sorted(p for r in rows for p in r if p >= live)
        to = dict(zip(high, holes))
        moves = list(to.items())
        rows = [[to.get(p, p) for p in r] for r in rows]
    res = {"k": [], "v": [], "table": [torch.tensor(r, dtype=torch.int32, device="cuda")
                                       for r in ([rows] if case["kind"] == "fork" else rows)]}
    for name in ("k", "v"):
        for t in getattr(cache, name):
            t = t.clone()
            for a, b in moves:
                t[b].copy_(t[a])
            res[name].append(t)
    return res


def _exact_attend(st):
    """Every sequence on its own over its whole context, head by head, in float64."""
    case = st["case"]
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G = H // KVH
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, t) in enumerate(zip(st["lens"], st["new"])):
        at = _tokens(st, b, 0, n)
        later = torch.arange(n, device="cuda")[None, :] > torch.arange(n - t, n, device="cuda")[:, None]
        for kv in range(KVH):
            k = st["k"].view(-1, KVH, D)[at, kv].double().t().contiguous()
            v = st["v"].view(-1, KVH, D)[at, kv].double()
            for h in range(kv * G, (kv + 1) * G):
                s = (st["q"][start:start + t, h].double() @ k) / math.sqrt(D)
                out[start:start + t, h] = torch.softmax(s.masked_fill(later, -math.inf), -1) @ v
        start += t
    return {"out": out}


def _exact_append(st):
    case = st["case"]
    H, KVH, D, page = case["H"], case["KVH"], case["D"], case["page"]
    x = st["qkv"].double()
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]
    c0, c1, s0, s1 = c[..., :D // 2], c[..., D // 2:], s[..., :D // 2], s[..., D // 2:]
    turned = torch.cat([a * c0 - b * s0, b * c1 + a * s1], -1)
    k, v = st["k"].double(), st["v"].double()
    table = st["table"].tolist()
    where = []
    for row, n, t in zip(table, st["lens"], st["new"]):
        where += [row[p // page] * page + p % page for p in range(n - t, n)]
    where = torch.tensor(where, device="cuda")
    k.view(-1, KVH, D).index_copy_(0, where, turned[:, H:H + KVH].contiguous())
    v.view(-1, KVH, D).index_copy_(0, where, x[:, H + KVH:].contiguous())
    return {"q": turned[:, :H], "k": k, "v": v}


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return _exact_pages(case, seed)
    st = prepare(case, seed)
    return _exact_attend(st) if case["kind"] == "attend" else _exact_append(st)
