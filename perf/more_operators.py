"""Several sequences of one prompt over a paged KV cache: beam search's selection
over beams and vocabulary, the reordering of the sequences' pages (forked,
copied, freed), the compaction of the pool, and attention of requests that
share a long prefix.

With `own` false, run() computes the operators in plain torch operations; with
`own` true it makes the calls of include/sejong_hip.h.  torch is imported
first: the library then runs on torch's HIP runtime and shares its devices and
pointers.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 4}  # SJ_F32, SJ_BF16
I32 = torch.int32


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a step of beam search with the byte vocabulary: 64 prompts of 4 beams, a row fits a wave: latency
        dict(name="select_bytes", kind="select", dtype="f32", groups=64, beams=4, vocab=257, ld=264, keep=4, power=0.0,
             ended=0.1, first=False),
        # one prompt, 8 beams of a large vocabulary, twice as many candidates as beams for the host's own bookkeeping
        dict(name="select_one", kind="select", dtype="f32", groups=1, beams=8, vocab=131072, ld=131072, keep=16, power=0.0,
             ended=0.0, first=False),
        # a batch of 48 prompts, a large odd vocabulary in bf16, ended beams, ranks normalised by length
        dict(name="select_batch", kind="select", dtype="bf16", groups=48, beams=8, vocab=50001, ld=50008, keep=8, power=0.6,
             ended=0.15, first=False),
        # the beams of 16 prompts change places: 64 requests of up to 4096 tokens
        dict(name="fork_beams", kind="fork", groups=16, beams=4, page=16, lo=40, hi=4096, spare=2048, gone=0.05),
        # a server's whole pool: 2000 requests, odd pages, 170000 pages
        dict(name="fork_pool", kind="fork", groups=400, beams=5, page=24, lo=100, hi=8000, spare=100000, gone=0.1),
        # behind a fork of 64 requests: the filled part of their last pages, in 8 layers of 4 heads of 64
        dict(name="copy_tails", kind="copy", dtype="bf16", layers=8, width=256, page=16, pages=512, count=64, whole=False),
        # behind a compaction: 600 whole pages, 8 layers of 8 heads of 64
        dict(name="copy_pages", kind="copy", dtype="bf16", layers=8, width=512, page=16, pages=1300, count=600, whole=True),
        # a pool of 2048 pages to half its size, 50 requests
        dict(name="compact_small", kind="compact", requests=50, page=16, pages=2048, after=1024, full=0.8),
        # a pool of 400000 pages to three quarters, 1000 requests
        dict(name="compact_large", kind="compact", requests=1000, page=16, pages=400001, after=300001, full=0.9),
        # 4 beams of one prompt near the end of the benchmark's model's context
        dict(name="shared_beams", kind="shared", dtype="bf16", groups=1, beams=4, per=1, pad=0, hq=6, hk=2, dim=64, page=16,
             lo=960, hi=960, tail=60, window=0),
        # 24 prompts of very different lengths, 5 fp32 beams each, odd pages, padded rows behind them
        dict(name="shared_ragged", kind="shared", dtype="f32", groups=24, beams=5, per=1, pad=3, hq=16, hk=4, dim=64, page=24,
             lo=24, hi=6000, tail=100, window=0),
        # a long document that 64 requests ask about, 128-wide heads
        dict(name="shared_document", kind="shared", dtype="bf16", groups=1, beams=64, per=1, pad=0, hq=32, hk=8, dim=128,
             page=64, lo=16384, hi=16384, tail=256, window=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["select", "select", "select", "fork", "copy", "compact", "shared", "shared", "shared"])
    if kind == "select":
        vocab = rng.choice([257, 257, _log(rng, 2, 2000), _log(rng, 2000, 150000), _log(rng, 30000, 150000)])
        beams = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32])
        groups = _log(rng, 1, max(1, min(512, 48 * 8 * 50001 // (vocab * beams))))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), groups=groups, beams=beams, vocab=vocab,
                    ld=vocab + rng.choice([0, 0, 1, 7]), keep=min(64, rng.choice([beams, beams, 2 * beams, beams + 1])),
                    power=rng.choice([0.0, 0.0, 0.6, 1.0]), ended=rng.choice([0.0, 0.1, 0.4]), first=rng.random() < 0.15)
    if kind == "fork":
        groups, beams = _log(rng, 1, 400), rng.choice([1, 2, 3, 4, 5])
        page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 256])
        hi = _log(rng, 2, max(2, min(8000, 150000 * page // (groups * beams))))
        return dict(kind=kind, groups=groups, beams=beams, page=page, lo=rng.choice([1, hi]), hi=hi,
                    spare=max(groups * beams, _log(rng, 16, 50000)), gone=rng.choice([0.0, 0.05, 0.3]))
    if kind == "copy":
        width, layers = rng.choice([1, 2, 4, 8]) * rng.choice([16, 32, 64, 80, 96, 128, 256]), rng.choice([1, 2, 6, 8, 12])
        page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256])
        count = _log(rng, 1, max(1, min(600, 600 * 16 * 8 * 512 // (page * layers * width * 2))))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), layers=layers, width=width, page=page,
                    pages=2 * count + rng.choice([0, 1, count // 2]), count=count, whole=rng.random() < 0.4)
    if kind == "compact":
        pages = _log(rng, 32, 400000)
        return dict(kind=kind, requests=_log(rng, 1, min(1000, pages // 8)), page=rng.choice([1, 8, 16, 24, 64, 256]),
                    pages=pages, after=max(8, int(pages * rng.uniform(0.3, 1.0))), full=rng.choice([0.1, 0.5, 0.9, 1.0]))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hk = rng.choice([1, 2, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([16, 32, 64, 64, 64, 80, 96, 128, 128, 256])
    groups, beams, per = rng.choice([1, 1, _log(rng, 1, 48)]), _log(rng, 1, 48), rng.choice([1, 1, 1, 2])
    rows = groups * beams * per
    most = 64 * 32 * 128 * 16384
    if dtype == "f32":
        most //= 8
    hi = _log(rng, 2, max(2, min(16384, most // (rows * hq * max(dim, 64)), 8 * 128 * 16384 // (groups * hk * dim))))
    lo = rng.choice([hi, _log(rng, 1, hi)])
    tail = _log(rng, 1, max(1, min(512, 64 * 256 * 8 * 128 // (rows * hk * dim))))
    return dict(kind=kind, dtype=dtype, groups=groups, beams=beams, per=per, pad=rng.choice([0, 0, 3]), hq=hq, hk=hk, dim=dim,
                page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]), lo=lo, hi=hi, tail=max(per, tail),
                window=rng.choice([0, 0, 0, 0, _log(rng, 1, 8192)]))


# ---------------------------------------------------------------- helpers

class _State:
    """What a case's program holds."""


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _spread(n, lo, hi):
    """n whole sizes between lo and hi, evenly spread over their logarithm."""
    at = (np.arange(n) + 0.5) / n
    return np.clip(np.rint(lo * (hi / lo) ** at), lo, hi).astype(np.int64)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _new(*shape, dtype=I32):
    return torch.empty(*shape, dtype=dtype, device=DEV)


# ---------------------------------------------------------------- prepare

def prepare(case, seed):
    s = _State()
    s.c, s.calls = case, None
    globals()["_prepare_" + case["kind"]](s, case, seed)
    return s


END = 1  # the token that ends a sequence


def _prepare_select(s, c, seed):
    """Logits with a few likely entries a row, as a trained model gives, and beams of like scores."""
    g = _gen(seed)
    n, V = c["groups"] * c["beams"], c["vocab"]
    s.dt = KINDS[c["dtype"]]
    x = torch.randn(n, c["ld"], generator=g, device=DEV) * 2.0
    likely = torch.randint(0, V, (n, 6), generator=g, device=DEV)
    x.scatter_add_(1, likely, torch.rand(n, 6, generator=g, device=DEV) * 12.0)
    s.x = x.to(s.dt)
    s.lengths = torch.randint(1, 200, (c["groups"], 1), generator=g, device=DEV).expand(-1, c["beams"]).reshape(-1).to(I32).contiguous()
    s.scores = -0.7 * s.lengths.float() + 1.5 * torch.randn(n, generator=g, device=DEV)
    s.ended = (torch.rand(n, generator=g, device=DEV) < c["ended"]).to(I32)
    if c["first"]:  # the first step: one beam of each prompt is alive
        s.scores.view(c["groups"], -1)[:, 1:] = -math.inf
        s.ended.zero_()
    m = c["groups"] * c["keep"]
    s.parents, s.tokens, s.lengths_after, s.ended_after = _new(m), _new(m), _new(m), _new(m)
    s.scores_after = _new(m, dtype=torch.float32)


def _beam_tables(c, rng):
    """Tables of groups of beams that share their first pages, as forks leave them, and the holders of every page."""
    P, G, B = c["page"], c["groups"], c["beams"]
    n = rng.permutation(_spread(G, c["lo"], c["hi"]))
    width = int(-(-c["hi"] // P)) + 1
    table, made = np.full((G * B, width), -1), 0
    for g in range(G):
        cols = int(-(-n[g] // P))
        full = int(n[g] // P)
        prompt = full * 3 // 4
        for b in range(B):
            row = table[g * B + b]
            same = 0
            if b:
                same = int(rng.integers(prompt, full + 1))
                row[:same] = table[g * B + int(rng.integers(0, b))][:same]
            row[same:cols] = np.arange(made, made + cols - same)
            made += cols - same
    cols, prompt = -(-n // P), n // P * 3 // 4
    pages = int((cols + (B - 1) * (cols - prompt)).sum()) + c["spare"]  # the most that the beams can have of their own
    names = rng.permutation(pages)
    held = table >= 0
    table[held] = names[table[held]]
    shared = np.maximum(np.bincount(table[held], minlength=pages) - 1, 0)
    for g in range(0, G, 7):  # some prompts are kept for requests to come
        shared[table[g * B, :int(n[g] // P * 3 // 4)]] += 1
    return np.repeat(n, B), table, shared, names[made:], pages


def _prepare_fork(s, c, seed):
    rng = np.random.default_rng(seed)
    G, B = c["groups"], c["beams"]
    lengths, table, shared, free, s.pages = _beam_tables(c, rng)
    parents = (np.arange(G)[:, None] * B + rng.integers(0, B, (G, B)))
    parents[rng.random(G) < c["gone"]] = -1  # prompts that are done
    s.requests, s.width = G * B, table.shape[1]
    s.parents, s.lengths, s.table, s.shared = _ints(parents.reshape(-1)), _ints(lengths), _ints(table), _ints(shared)
    s.free = _ints(np.concatenate([np.full(s.pages - len(free), -1), free]))
    s.head = _ints([s.pages - len(free)])
    s.table_after, s.lengths_after = torch.empty_like(s.table), torch.empty_like(s.lengths)
    s.shared_after, s.free_after = torch.empty_like(s.shared), torch.empty_like(s.free)
    s.copies, s.summary = _new(s.requests, 3), _new(4)


def _prepare_copy(s, c, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    s.dt = KINDS[c["dtype"]]
    rows = c["pages"] * c["page"]
    s.k, s.v = (_new(c["layers"], rows, c["width"], dtype=s.dt).normal_(generator=g) for _ in range(2))
    order = rng.permutation(c["pages"])[:2 * c["count"]]
    slots = np.full(c["count"], c["page"]) if c["whole"] else rng.integers(1, c["page"] + 1, c["count"])
    copies = np.stack([order[:c["count"]], order[c["count"]:], slots], 1)
    if not c["whole"]:
        copies[rng.random(c["count"]) < 0.1] = [-1, -1, 0]  # these kept their page
    s.copies = _ints(copies)


def _compact_sizes(c):
    """How many pages the requests hold: never more than the smaller pool has."""
    return max(1, int(c["after"] * c["full"]))


def _prepare_compact(s, c, seed):
    rng = np.random.default_rng(seed)
    P, R, used = c["page"], c["requests"], _compact_sizes(c)
    share = _spread(R, 8, 64)  # requests of up to eight times the others' pages
    cols = rng.permutation(used * share // share.sum())
    s.width = int(cols.max()) + 2
    names = rng.permutation(c["pages"])
    table = np.full((R, s.width), -1)
    table[np.arange(s.width)[None, :] < cols[:, None]] = names[:int(cols.sum())]
    shared = np.zeros(c["pages"], np.int64)
    for r in range(1, R, 2):  # these have the beginning of the request before
        m = int(min(cols[r], cols[r - 1]) // 2)
        table[r, :m] = table[r - 1, :m]
        shared[table[r, :m]] += 1
    lengths = np.maximum(cols * P - rng.integers(0, P, R), 0)
    held = np.zeros(c["pages"], bool)
    held[table[table >= 0]] = True
    free = rng.permutation(np.nonzero(~held)[0])
    s.lengths, s.table, s.shared = _ints(np.where(cols > 0, lengths, 0)), _ints(table), _ints(shared)
    s.free = _ints(np.concatenate([np.full(c["pages"] - len(free), -1), free]))
    s.head = _ints([c["pages"] - len(free)])
    s.capacity = c["pages"] - c["after"]
    s.table_after, s.shared_after, s.free_after = torch.empty_like(s.table), torch.empty_like(s.shared), torch.empty_like(s.free)
    s.copies, s.summary = _new(s.capacity, 3), _new(4)


def _shared_sizes(c):
    """Shared positions of every group (whole pages, as a prefix cache has them) and the own tokens of every request."""
    P = c["page"]
    prefix = np.maximum(_spread(c["groups"], c["lo"], c["hi"]) // P, 0) * P
    tails = _spread(c["groups"] * c["beams"], c["per"], c["tail"])
    return prefix, tails


def _prepare_shared(s, c, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    s.dt, P, G, B, per = KINDS[c["dtype"]], c["page"], c["groups"], c["beams"], c["per"]
    prefix, tails = _shared_sizes(c)
    prefix, tails = rng.permutation(prefix), rng.permutation(tails)
    lead, mine = prefix // P, -(-tails // P)
    s.requests, s.width = G * B, int(lead.max() + mine.max())
    s.pages = int(lead.sum() + mine.sum()) + 5
    names = rng.permutation(s.pages)
    table, made = np.full((G * B, s.width), -1), 0
    for q in range(G):
        first = names[made:made + lead[q]]
        made += int(lead[q])
        for r in range(q * B, (q + 1) * B):
            table[r, :lead[q]] = first
            table[r, lead[q]:lead[q] + mine[r]] = names[made:made + mine[r]]
            made += int(mine[r])
    # the last `per` tokens of each request ask
    positions = (np.repeat(prefix, B) + tails)[:, None] - per + np.arange(per)[None, :]
    s.prefix, s.group_starts = _ints(prefix), _ints(np.arange(G + 1) * B)
    s.starts, s.table = _ints(np.arange(G * B + 1) * per), _ints(table)
    s.positions = _ints(np.concatenate([positions.reshape(-1), np.full(c["pad"], -1)]))
    s.owners = _ints(np.concatenate([np.repeat(np.arange(G * B), per), np.full(c["pad"], -1)]))
    s.rows = G * B * per + c["pad"]
    w = c["hk"] * c["dim"]
    s.k, s.v = (_new(s.pages * P, w, dtype=s.dt).normal_(generator=g) for _ in range(2))
    s.q = (1.5 * torch.randn(s.rows, c["hq"] * c["dim"], generator=g, device=DEV)).to(s.dt)
    s.o = torch.zeros_like(s.q)
    s.lse = torch.zeros(s.rows, c["hq"], device=DEV)
    s.own_most = int(tails.max())


# -------------------------------------------------------------------- run

def run(s):
    if own:
        if s.calls is None:
            s.calls = _Calls()
            s.result = globals()["_own_" + s.c["kind"]](s, s.calls)
        for fn, args in s.calls.all:
            s.calls.check(fn(*args))
        return s.result
    return globals()["_plain_" + s.c["kind"]](s)


class _Calls:
    """The C ABI calls of a pass with their arguments, as a compiled caller has
    them: a pass then costs the calls themselves, not Python's packing."""

    def __init__(self):
        from sejong_amd import _native as N
        self.lib, self.check, self.all = N.load(), N.check, []

    def add(self, name, *args):
        fn = getattr(self.lib, name)
        out = []
        for a, t in zip(args, fn.argtypes):
            out.append(t(a.data_ptr()) if isinstance(a, torch.Tensor) else a if isinstance(a, t) else t(a))
        self.all.append((fn, tuple(out)))

    def scratch(self, name, *sizes):
        """The workspace of a call, kept by the program."""
        return torch.empty(max(int(getattr(self.lib, name)(*sizes)), 256), dtype=torch.uint8, device=DEV)


# select

def _own_select(s, a):
    c = s.c
    s.work = a.scratch("sj_beam_select_workspace_bytes", c["groups"], c["beams"], c["vocab"], c["keep"])
    a.add("sj_beam_select", None, s.x, CODES[c["dtype"]], c["ld"], c["groups"], c["beams"], c["vocab"], s.scores, s.lengths,
          s.ended, END, c["power"], c["keep"], s.parents, s.tokens, s.scores_after, s.lengths_after, s.ended_after, s.work,
          s.work.numel())
    return dict(parents=s.parents, tokens=s.tokens, scores=s.scores_after, lengths=s.lengths_after, ended=s.ended_after)


def _plain_select(s):
    c, G, B, V, K = s.c, s.c["groups"], s.c["beams"], s.c["vocab"], s.c["keep"]
    n, k = G * B, min(K, V)
    x = s.x[:, :V].float()
    # whole keys in the order of the values, the lowest index first among equals
    bits = (x + 0.0).view(I32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    keys = order * (1 << 20) - torch.arange(V, device=DEV)
    best = (-torch.topk(keys, k, dim=-1).values) & ((1 << 20) - 1)
    # totals in 64 bits: those of different beams may lie next to each other
    x = x.double()
    m = x.amax(-1, keepdim=True)
    total = s.scores.double()[:, None] + (x.gather(1, best) - (m + (x - m).exp().sum(-1, keepdim=True).log()))
    ended = (s.ended != 0)[:, None]
    only = torch.arange(k, device=DEV)[None, :] == 0
    total = torch.where(ended, torch.where(only, s.scores.double()[:, None], -math.inf), total)
    best = torch.where(ended & only, END, best)
    length = s.lengths.long()[:, None] + (~ended).long()
    rank = total / length.clamp(min=1).double().pow(c["power"]) if c["power"] else total
    # of the candidates in the order of beam and token, those of the highest ranks
    flat = (torch.arange(n, device=DEV)[:, None] % B) * V + best
    flat, rank, total = (t.view(G, -1) for t in (flat, rank, total))
    at = flat.argsort(-1)
    at = at.gather(1, rank.gather(1, at).sort(dim=-1, descending=True, stable=True).indices)[:, :K]
    if at.shape[1] < K:
        at = torch.cat([at, at[:, :1].expand(-1, K - at.shape[1])], 1)
    some = (total.gather(1, at) > -math.inf) & (torch.arange(K, device=DEV) < B * k)
    flat, total = flat.gather(1, at), total.gather(1, at)
    parent = flat // V + torch.arange(G, device=DEV)[:, None] * B
    token = flat % V
    done = (s.ended.long()[parent] != 0) | (token == END)

    def fill(t, none):
        return torch.where(some, t, none).reshape(-1)

    return dict(parents=fill(parent, -1).to(I32), tokens=fill(token, -1).to(I32), scores=fill(total, -math.inf).float(),
                lengths=fill(s.lengths.long()[parent] + (s.ended.long()[parent] == 0), 0).to(I32),
                ended=fill(done.long(), 1).to(I32))


# fork

def _own_fork(s, a):
    c = s.c
    s.work = a.scratch("sj_paged_fork_workspace_bytes", s.requests, s.requests, s.pages)
    a.add("sj_paged_fork", None, s.parents, s.requests, s.table, s.width, s.lengths, s.requests, c["page"], s.pages, s.shared,
          s.free, s.free.numel(), s.head, s.table_after, s.lengths_after, s.shared_after, s.free_after, s.copies, s.summary,
          s.work, s.work.numel())
    return dict(table=s.table_after, lengths=s.lengths_after, shared=s.shared_after, free=s.free_after, copies=s.copies,
                summary=s.summary)


def _plain_fork(s):
    P, R, dev = s.c["page"], s.requests, DEV
    n, parents = s.lengths.long(), s.parents.long()
    live = parents >= 0
    p = parents.clamp(min=0)
    child = torch.arange(R, device=dev)
    count = torch.zeros(R + 1, dtype=torch.long, device=dev).index_add(0, torch.where(live, p, R), torch.ones_like(p))[:R]
    first = torch.full((R + 1,), R, device=dev).scatter_reduce(0, torch.where(live, p, R), child, "amin")[:R]
    full, tail = n // P, n % P
    page = s.table.long().gather(1, full.clamp(max=s.width - 1)[:, None])[:, 0]  # the page that is not full
    alone = s.shared.long()[page.clamp(min=0)] <= 0
    # the children that get a page of their own, from the free list in their order
    takes = live & (tail[p] > 0) & ((first[p] != child) | ~alone[p])
    head = s.head.long()[0]
    place = torch.cumsum(takes.long(), 0) - 1
    fresh = s.free.long()[(head + place).clamp(0, s.free.numel() - 1)]
    col = torch.arange(s.width, device=dev)[None, :]
    table = torch.where(live[:, None] & (col < ((n + P - 1) // P)[p][:, None]), s.table.long()[p], -1)
    table = torch.where(takes[:, None] & (col == full[p][:, None]), fresh[:, None], table)
    copies = torch.where(takes[:, None], torch.stack([page[p], fresh, tail[p]], 1), torch.tensor([-1, -1, 0], device=dev))
    # the pages' holders after the step; those without any go back, the highest first in the list
    change = torch.where(col < full[:, None], (count - 1)[:, None], 0)
    change = torch.where((col == full[:, None]) & (tail > 0)[:, None],
                         torch.where(alone & (count > 0), 0, -1)[:, None], change)
    held = torch.where((col < ((n + P - 1) // P)[:, None]), s.table.long(), s.pages)
    shared = torch.cat([s.shared.long(), s.shared.new_zeros(1).long()]).index_add(0, held.reshape(-1), change.reshape(-1))
    shared = shared[:s.pages]
    back = shared < 0
    head = head + takes.long().sum()
    place = torch.where(back, head - torch.cumsum(back.long(), 0), s.free.numel())
    free = torch.cat([s.free.long(), s.free.new_zeros(1).long()])
    free = free.index_copy(0, place, torch.arange(s.pages, device=dev))[:-1]
    summary = torch.stack([takes.long().sum(), head - back.long().sum(), torch.zeros_like(head), back.long().sum()])
    return dict(table=table.to(I32), lengths=torch.where(live, n[p], 0).to(I32), shared=torch.where(back, 0, shared).to(I32),
                free=free.to(I32), copies=copies.to(I32), summary=summary.to(I32))


# copy

def _own_copy(s, a):
    c = s.c
    a.add("sj_paged_copy", None, s.k, s.v, c["width"], CODES[c["dtype"]], c["layers"], s.k.stride(0), c["pages"], c["page"],
          c["width"], s.copies, c["count"])
    return dict(k=s.k, v=s.v)


def _plain_copy(s):
    P = s.c["page"]
    j = torch.arange(P, device=DEV)
    from_, to, slots = (t.long() for t in s.copies.unbind(1))
    moved = (j[None, :] < slots[:, None]) & (from_ >= 0)[:, None]
    at = (to[:, None] * P + j)[moved]
    of = (from_[:, None] * P + j)[moved]
    for cache in (s.k, s.v):
        cache[:, at] = cache[:, of]
    return dict(k=s.k, v=s.v)


# compact

def _own_compact(s, a):
    c = s.c
    s.work = a.scratch("sj_paged_compact_workspace_bytes", c["pages"], c["pages"])
    a.add("sj_paged_compact", None, s.table, s.width, s.lengths, c["requests"], c["page"], c["pages"], c["after"], s.shared,
          s.free, s.free.numel(), s.head, s.table_after, s.shared_after, s.free_after, s.copies, s.capacity, s.summary, s.work,
          s.work.numel())
    return dict(table=s.table_after, shared=s.shared_after, free=s.free_after, copies=s.copies, summary=s.summary)


def _plain_compact(s):
    c, N, dev = s.c, s.c["pages"], DEV
    head = s.head.long()[0]
    at = torch.arange(s.free.numel(), device=dev)
    on_list = at >= head
    free = s.free.long()
    is_free = torch.zeros(N + 1, dtype=torch.bool, device=dev).index_fill(0, torch.where(on_list, free, N), True)[:N]
    page = torch.arange(N, device=dev)
    moves = (page >= c["after"]) & ~is_free
    below = on_list & (free < c["after"])
    nmoves, nbelow = moves.long().sum(), below.long().sum()
    # the j-th page that moves gets the j-th free page below
    order = torch.cumsum(moves.long(), 0) - 1
    place = torch.cumsum(below.long(), 0) - 1
    target = torch.zeros(N + 1, dtype=torch.long, device=dev).index_copy(0, torch.where(below, place, N), free)
    to = torch.where(moves, target[order.clamp(min=0)], page)
    col = torch.arange(s.width, device=dev)[None, :]
    used = col < ((s.lengths.long() + c["page"] - 1) // c["page"])[:, None]
    t = s.table.long()
    table = torch.where(used & (t >= 0) & (t < N), to[t.clamp(0, N - 1)], -1)
    shared = torch.where(page >= c["after"], 0, s.shared.long())
    shared = torch.cat([shared, shared[:1]]).index_copy(0, torch.where(moves, to, N), s.shared.long())[:N]
    left = below & (place >= nmoves)
    after = torch.full((s.free.numel() + 1,), -1, dtype=torch.long, device=dev)
    after = after.index_copy(0, torch.where(left, s.free.numel() - nbelow + place, s.free.numel()), free)[:-1]
    copies = torch.tensor([-1, -1, 0], device=dev).repeat(s.capacity + 1, 1)
    copies = copies.index_copy(0, torch.where(moves, order, s.capacity), torch.stack([page, to, torch.full_like(page, c["page"])], 1))
    summary = torch.stack([nmoves, s.free.numel() - nbelow + nmoves, torch.zeros_like(nmoves), nbelow - nmoves])
    return dict(table=table.to(I32), shared=shared.to(I32), free=after.to(I32), copies=copies[:-1].to(I32),
                summary=summary.to(I32))


# shared

def _own_shared(s, a):
    c, w = s.c, s.c["hk"] * s.c["dim"]
    s.work = a.scratch("sj_paged_attention_shared_workspace_bytes", s.rows, c["hq"], c["hk"], c["dim"], c["groups"])
    a.add("sj_paged_attention_shared", None, s.q, c["hq"] * c["dim"], s.k, s.v, w, CODES[c["dtype"]], s.pages, c["page"],
          s.table, s.width, s.requests, s.owners, s.positions, s.rows, s.starts, s.group_starts, s.prefix, c["groups"],
          c["hq"], c["hk"], c["dim"], c["window"], s.o, c["hq"] * c["dim"], s.lse, s.work, s.work.numel())
    return dict(o=s.o, lse=s.lse)


def _plain_shared(s):
    """The prefix's keys once for all rows of a group, and every row's own."""
    c, P, D, G = s.c, s.c["page"], s.c["dim"], s.c["groups"]
    hk, g, n = c["hk"], c["hq"] // c["hk"], c["beams"] * c["per"]
    rows = G * n
    q = s.q[:rows].float() * D ** -0.5
    pos = s.positions.long()[:rows]
    prefix = s.prefix.long()

    def seen_of(j, upto):
        seen = j < upto
        return seen & (j > pos[:, None] - c["window"]) if c["window"] else seen

    # [group][head][rows x heads of the group] against the prefix, [row][head][heads of the group] against the rest
    lead = int(-(-c["hi"] // P) * P)
    j = torch.arange(lead, device=DEV)
    page = s.table.long()[s.group_starts.long()[:-1]][:, (j // P).clamp(max=s.width - 1)]
    slot = torch.where((j[None, :] < prefix[:, None]) & (page >= 0), page * P + j % P, 0)
    kp, vp = (t[slot].float().view(G, lead, hk, D).transpose(1, 2).contiguous() for t in (s.k, s.v))
    qg = q.view(G, n, hk, g, D).transpose(1, 2).reshape(G, hk, n * g, D)
    sp = torch.matmul(qg, kp.transpose(2, 3).contiguous()).view(G, hk, n, g, lead).transpose(1, 2).reshape(rows, hk, g, lead)
    seen = seen_of(j[None, :], prefix.repeat_interleave(n)[:, None])
    sp = sp.masked_fill(~seen[:, None, None, :], -math.inf)
    i = prefix.repeat_interleave(n)[:, None] + torch.arange(s.own_most, device=DEV)[None, :]
    page = s.table.long()[s.owners.long()[:rows]].gather(1, (i // P).clamp(max=s.width - 1))
    seen = seen_of(i, pos[:, None] + 1) & (page >= 0)
    slot = torch.where(seen, page * P + i % P, 0)
    ko, vo = (t[slot].float().view(rows, -1, hk, D).transpose(1, 2).contiguous() for t in (s.k, s.v))
    so = torch.matmul(q.view(rows, hk, g, D), ko.transpose(2, 3).contiguous()).masked_fill(~seen[:, None, None, :], -math.inf)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = (sp - top).exp(), (so - top).exp()
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    pg = sp.view(G, n, hk, g, lead).transpose(1, 2).reshape(G, hk, n * g, lead)
    o = torch.matmul(pg, vp).view(G, hk, n, g, D).transpose(1, 2).reshape(rows, hk, g, D) + torch.matmul(so, vo)
    o, lse = o / total, top + total.log()
    out = dict(o=torch.zeros_like(s.q), lse=torch.zeros_like(s.lse))  # padded rows are left as they were
    out["o"][:rows], out["lse"][:rows] = o.reshape(rows, -1).to(s.dt), lse.reshape(rows, -1)
    return out


# ------------------------------------------------------------------- work

def work(c):
    kind = c["kind"]
    if kind == "select":
        n, size = c["groups"] * c["beams"], 4 if c["dtype"] == "f32" else 2
        live = n * (1.0 - c["ended"])
        return dict(bytes=int(live * c["vocab"] * size) + 12 * n + 20 * c["groups"] * c["keep"],
                    flops=int(live * c["vocab"] * 4))
    if kind == "fork":
        R, P = c["groups"] * c["beams"], c["page"]
        held = int((-(-_spread(c["groups"], c["lo"], c["hi"]) // P)).sum()) * c["beams"]
        width, pages = int(-(-c["hi"] // P)) + 1, held // 2 + c["spare"]
        return dict(bytes=4 * (held + R * width + 6 * R + 4 * pages), flops=0)
    if kind == "copy":
        size = 4 if c["dtype"] == "f32" else 2
        slots = c["count"] * (c["page"] if c["whole"] else 0.9 * (c["page"] + 1) / 2)
        return dict(bytes=int(4 * slots * c["layers"] * c["width"] * size) + 12 * c["count"], flops=0)
    if kind == "compact":
        used = _compact_sizes(c)
        return dict(bytes=4 * (2 * used + c["requests"] + 4 * c["pages"] + 3 * (c["pages"] - c["after"])), flops=0)
    prefix, tails = _shared_sizes(c)
    size, window, n = 4 if c["dtype"] == "f32" else 2, c["window"] or 1 << 40, c["beams"] * c["per"]
    rows = c["groups"] * n
    keys = int(np.minimum(prefix, window).sum() + np.minimum(tails, window).sum())
    seen = int(np.minimum(np.repeat(prefix, c["beams"]) + tails, window).sum()) * c["per"]
    return dict(bytes=2 * keys * c["hk"] * c["dim"] * size + rows * c["hq"] * (2 * c["dim"] * size + 4),
                flops=4 * seen * c["hq"] * c["dim"])


# ------------------------------------------------------------------ exact

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](s, case)


def _exact_select(s, c):
    B, V, K = c["beams"], c["vocab"], c["keep"]
    scores, lengths, ended = s.scores.double(), s.lengths.tolist(), s.ended.tolist()
    out = dict(parents=[], tokens=[], scores=[], lengths=[], ended=[])
    for g in range(c["groups"]):
        total = torch.full((B, V), -math.inf, dtype=torch.float64, device=DEV)
        rank = total.clone()
        for b in range(B):
            r = g * B + b
            if ended[r]:
                total[b, END] = scores[r]
                rank[b, END] = scores[r] / max(lengths[r], 1) ** c["power"]
            else:
                total[b] = scores[r] + torch.log_softmax(s.x[r, :V].double(), -1)
                rank[b] = total[b] / (lengths[r] + 1) ** c["power"]
        best = torch.sort(rank.view(-1), descending=True, stable=True).indices[:K].tolist()
        total = total.view(-1)
        for i in range(K):
            t = float(total[best[i]]) if i < len(best) else -math.inf
            if t == -math.inf:
                for key, none in zip(("parents", "tokens", "scores", "lengths", "ended"), (-1, -1, t, 0, 1)):
                    out[key].append(none)
                continue
            r, v = g * B + best[i] // V, best[i] % V
            out["parents"].append(r)
            out["tokens"].append(v)
            out["scores"].append(t)
            out["lengths"].append(lengths[r] + (0 if ended[r] else 1))
            out["ended"].append(int(ended[r] != 0 or v == END))
    return {k: np.array(v, np.float64 if k == "scores" else np.int32) for k, v in out.items()}


def _exact_fork(s, c):
    P, R = c["page"], s.requests
    table, lengths, parents = s.table.cpu().numpy(), s.lengths.cpu().numpy(), s.parents.cpu().numpy()
    shared, free, head = s.shared.cpu().numpy().astype(np.int64), s.free.cpu().numpy().copy(), int(s.head)
    holders = shared + 1
    before = shared.copy()
    after, lengths_after, copies = np.full_like(table, -1), np.zeros(R, np.int32), np.tile([-1, -1, 0], (R, 1))
    heir = {}
    for r in range(R):  # the rows let go of their pages
        cols = -(-int(lengths[r]) // P)
        holders[table[r, :cols]] -= 1
    taken = 0
    for i, r in enumerate(parents):
        if r < 0:
            continue
        n = int(lengths[r])
        full, cols = n // P, -(-n // P)
        after[i, :cols] = table[r, :cols]
        lengths_after[i] = n
        if cols > full:
            if r in heir or before[table[r, full]] > 0:
                after[i, full] = free[head + taken]
                copies[i] = [table[r, full], free[head + taken], n % P]
                taken += 1
            heir.setdefault(r, i)
        holders[after[i, :cols]] += 1
    at = head + taken
    given = (s.shared.cpu().numpy() >= 0) & (holders == 0)
    was_free = np.zeros(s.pages, bool)
    was_free[free[head:]] = True  # free pages have no holder to lose
    back = np.nonzero(given & ~was_free)[0]
    holders[free[head + taken:]] = 1
    free[at - len(back):at] = back[::-1]
    shared_after = np.maximum(holders - 1, 0)
    taken_pages = copies[copies[:, 0] >= 0][:, 1]
    shared_after[taken_pages] = 0
    return dict(table=after, lengths=lengths_after, shared=shared_after.astype(np.int32), free=free,
                copies=copies.astype(np.int32), summary=np.array([taken, at - len(back), 0, len(back)], np.int32))


def _exact_copy(s, c):
    P = c["page"]
    out = dict(k=s.k.clone(), v=s.v.clone())
    for f, t, n in s.copies.tolist():
        if f >= 0:
            for cache in (out["k"], out["v"]):
                cache[:, t * P:t * P + n] = cache[:, f * P:f * P + n]
    return out


def _exact_compact(s, c):
    free, head, after = s.free.cpu().numpy(), int(s.head), c["after"]
    rest = free[head:].tolist()
    listed_ = set(rest)
    below = [p for p in rest if p < after]
    moves = [p for p in range(after, c["pages"]) if p not in listed_]
    to = dict(zip(moves, below))
    table, lengths = s.table.cpu().numpy(), s.lengths.cpu().numpy()
    out = np.full_like(table, -1)
    for r in range(len(lengths)):
        for col in range(-(-int(lengths[r]) // c["page"])):
            out[r, col] = to.get(int(table[r, col]), table[r, col])
    shared = s.shared.cpu().numpy()
    shared_after = shared.copy()
    shared_after[after:] = 0
    for p, t in to.items():
        shared_after[t] = shared[p]
    left = below[len(moves):]
    free_after = np.full(len(free), -1, np.int32)
    if left:
        free_after[len(free) - len(left):] = left
    copies = np.tile([-1, -1, 0], (s.capacity, 1)).astype(np.int32)
    for i, p in enumerate(moves):
        copies[i] = [p, to[p], c["page"]]
    return dict(table=out, shared=shared_after, free=free_after, copies=copies,
                summary=np.array([len(moves), len(free) - len(left), 0, len(left)], np.int32))


def _exact_shared(s, c):
    P, D, hk, g = c["page"], c["dim"], c["hk"], c["hq"] // c["hk"]
    o = torch.zeros(s.rows, hk, g, D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s.rows, hk, g, dtype=torch.float64, device=DEV)
    owners, positions = s.owners.tolist(), s.positions.tolist()
    for r in range(s.rows):
        if positions[r] < 0:
            continue
        j = torch.arange(max(0, positions[r] + 1 - c["window"]) if c["window"] else 0, positions[r] + 1, device=DEV)
        slot = s.table[owners[r]].long()[j // P] * P + j % P
        k, v = (t[slot].double().view(-1, hk, D).transpose(0, 1).contiguous() for t in (s.k, s.v))
        score = torch.matmul(k, s.q[r].double().view(hk, g, D).transpose(1, 2).contiguous()) / math.sqrt(D)
        lse[r] = torch.logsumexp(score, 1)
        o[r] = torch.matmul(torch.softmax(score, 1).transpose(1, 2).contiguous(), v)
    return dict(o=o.reshape(s.rows, -1), lse=lse.reshape(s.rows, -1))
