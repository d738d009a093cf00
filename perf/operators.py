"""One decoding step of many sequences over a paged KV cache, and what is said
about its tokens: the step's plan (block tables, positions, slots), rotary
positions and the cache append, attention over the pages, and log
probabilities of given tokens with entropy, alternatives and gradient.

With `own` false, run() computes the operators in plain torch operations; with
`own` true it makes the calls of include/sejong_hip.h.  torch is imported
first: the library then runs on torch's HIP runtime and shares its devices and
pointers.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 4}  # SJ_F32, SJ_BF16
INTERLEAVED, HALF = 0, 1
UNSCALED, LINEAR, BASE, PARTS = 0, 1, 2, 3


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a decoding step of 64 running requests, one new token each: pure latency
        dict(name="plan_decode", kind="plan", requests=64, page=16, lo=1, hi=4096, new_lo=1, new_hi=1, pad=0),
        # prompts arrive: 1500 requests with up to 2000 new tokens each, an odd page size, padded rows behind them
        dict(name="plan_prompts", kind="plan", requests=1500, page=24, lo=1, hi=8000, new_lo=1, new_hi=2000, pad=1000),
        # training: query and key heads of 16384 tokens inside the q|k|v buffer, half layout, positions of a long
        # context with frequencies scaled by parts
        dict(name="rope_half_bf16", kind="rope", dtype="bf16", rows=16384, heads=20, dim=64, rot=64, layout=HALF,
             scaling=PARTS, span=131072, inverse=False),
        # its gradient: fp32, interleaved pairs, inverse rotation, 40 of 96 columns rotated, an odd number of rows
        dict(name="rope_back_f32", kind="rope", dtype="f32", rows=4099, heads=6, dim=96, rot=40, layout=INTERLEAVED,
             scaling=UNSCALED, span=2048, inverse=True),
        # decoding: 100 new tokens rotated, their keys and values written to the cache's slots, 4 padded rows
        dict(name="append_decode", kind="append", dtype="bf16", rows=104, pad=4, hq=16, hk=4, dim=64, rot=64,
             layout=INTERLEAVED, scaling=UNSCALED, span=4096),
        # interactive use: one request of the benchmark's model near the end of its context
        dict(name="attend_one", kind="attend", dtype="bf16", requests=1, per=1, pad=0, hq=6, hk=2, dim=64, page=16,
             lo=1000, hi=1000, window=0),
        # a server's batch: 45 requests of very different lengths, odd pages, three padded rows
        dict(name="attend_ragged", kind="attend", dtype="bf16", requests=45, per=1, pad=3, hq=16, hk=4, dim=64, page=24,
             lo=1, hi=6000, window=0),
        # the largest: 64 long requests with 128-wide heads, more keys than the last-level cache holds
        dict(name="attend_long", kind="attend", dtype="bf16", requests=64, per=1, pad=0, hq=32, hk=8, dim=128, page=64,
             lo=4000, hi=16384, window=0),
        # the fp32 model's form with a sliding window, two draft tokens a request
        dict(name="attend_f32_window", kind="attend", dtype="f32", requests=33, per=2, pad=0, hq=4, hk=2, dim=32, page=16,
             lo=10, hi=2000, window=700),
        # byte vocabulary: scores, entropy, alternatives and their gradient for 4096 trained tokens
        dict(name="score_bytes", kind="score", dtype="f32", rows=4096, vocab=257, ld=264, top=5, back=True),
        # a decoding step's answers: few rows of a large vocabulary, 20 alternatives
        dict(name="score_decode", kind="score", dtype="f32", rows=32, vocab=131072, ld=131072, top=20, back=False),
        # training on a large odd vocabulary in bf16
        dict(name="score_train", kind="score", dtype="bf16", rows=2048, vocab=50001, ld=50008, top=8, back=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "append", "attend", "attend", "attend", "score", "score"])
    if kind == "plan":
        requests = _log(rng, 1, 4000)
        if rng.random() < 0.5:
            lo = hi = rng.randint(1, 2)
        else:
            lo, hi = 1, max(2, min(4000, _log(rng, 2, 4000), 1200000 // requests))
        return dict(kind=kind, requests=requests, page=rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 256]), lo=1,
                    hi=_log(rng, 2, 8000), new_lo=lo, new_hi=hi, pad=rng.choice([0, 0, _log(rng, 1, 2000)]))
    if kind == "rope":
        dim = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        heads = _log(rng, 1, 40)
        rows = _log(rng, 1, max(1, min(65536, 16384 * 20 * 64 // (heads * dim))))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), rows=rows, heads=heads, dim=dim, rot=rot,
                    layout=rng.choice([INTERLEAVED, HALF]), scaling=rng.choice([UNSCALED, LINEAR, BASE, PARTS]),
                    span=_log(rng, 512, 1 << 20), inverse=rng.random() < 0.5)
    if kind == "append":
        dim = rng.choice([16, 32, 64, 64, 96, 128, 256])
        hk = rng.choice([1, 2, 4, 8])
        rows = _log(rng, 1, 2000)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), rows=rows, pad=rng.randint(0, rows // 4),
                    hq=hk * rng.choice([1, 2, 3, 4, 8]), hk=hk, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    layout=rng.choice([INTERLEAVED, HALF]), scaling=rng.choice([UNSCALED, LINEAR, BASE, PARTS]),
                    span=_log(rng, 512, 1 << 20))
    if kind == "attend":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        hk = rng.choice([1, 2, 2, 4, 8])
        dim = rng.choice([16, 32, 64, 64, 64, 80, 96, 128, 128, 256])
        requests, per = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 4])
        size = 4 if dtype == "f32" else 2
        hi = _log(rng, 2, max(2, min(16384, (1 << 31) // (requests * per * hk * dim * 2 * size))))
        lo = rng.choice([hi, _log(rng, 1, hi)])
        return dict(kind=kind, dtype=dtype, requests=requests, per=per, pad=rng.choice([0, 0, 3]),
                    hq=hk * rng.choice([1, 2, 3, 4, 7, 8, 16, 20]), hk=hk, dim=dim,
                    page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]), lo=lo, hi=hi,
                    window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))
    vocab = rng.choice([257, 257, _log(rng, 2, 2000), _log(rng, 2000, 150000), _log(rng, 30000, 150000)])
    rows = _log(rng, 1, max(1, min(16384, 2048 * 50001 // vocab)))
    return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), rows=rows, vocab=vocab, ld=vocab + rng.choice([0, 0, 1, 7]),
                top=min(vocab, rng.choice([1, 2, 5, 8, 20, 32])), back=rng.random() < 0.5)


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


def _plan_sizes(c):
    lengths, counts = _spread(c["requests"], c["lo"], c["hi"]), _spread(c["requests"], c["new_lo"], c["new_hi"])
    return lengths, counts


def _capacity(c):
    return int(_plan_sizes(c)[1].sum()) + c["pad"]


# ---------------------------------------------------------------- prepare

def prepare(case, seed):
    s = _State()
    s.c, s.calls = case, None
    globals()["_prepare_" + case["kind"]](s, case, seed)
    return s


def _prepare_plan(s, c, seed):
    """Requests with pages in hand, in a pool whose other pages are free."""
    rng = np.random.default_rng(seed)
    lengths, counts = _plan_sizes(c)
    lengths, counts = rng.permutation(lengths), rng.permutation(counts)
    counts[rng.random(len(counts)) < 0.05] = 0  # requests that wait
    P = c["page"]
    have, want = -(-lengths // P), -(-(lengths + counts) // P)
    s.width = int(-(-(c["hi"] + c["new_hi"]) // P)) + 1
    s.pages = int(want.sum()) + 64
    order = rng.permutation(s.pages)
    table = np.full((c["requests"], s.width), -1)
    mask = np.arange(s.width)[None, :] < have[:, None]
    table[mask] = order[:int(have.sum())]
    s.lengths, s.counts, s.table0 = _ints(lengths), _ints(counts), _ints(table)
    s.free = _ints(np.concatenate([np.full(3, -1), order[int(have.sum()):]]))  # three are taken already
    s.head = _ints([3])
    s.table = s.table0.clone()
    s.rows = _capacity(c)
    s.starts = torch.empty(c["requests"] + 1, dtype=torch.int32, device=DEV)
    s.positions, s.slots, s.owners = (torch.empty(s.rows, dtype=torch.int32, device=DEV) for _ in range(3))
    s.after = torch.empty_like(s.lengths)
    s.summary = torch.empty(4, dtype=torch.int32, device=DEV)


def _scaling(c):
    return dict(theta=10000.0, kind=c["scaling"], factor=8.0, context=8192.0, fast=32.0, slow=1.0)


def _amplitude(c):
    return 0.1 * math.log(8.0) + 1.0 if c["scaling"] == PARTS else 1.0


def _prepare_rope(s, c, seed):
    """The rotated columns lie in a wider buffer (q|k of a q|k|v row)."""
    g = _gen(seed)
    s.dt = KINDS[c["dtype"]]
    s.ld = (c["heads"] + 4) * c["dim"]
    s.x = torch.randn(c["rows"], s.ld, generator=g, device=DEV).to(s.dt)
    s.positions = torch.randint(0, c["span"], (c["rows"],), generator=g, device=DEV, dtype=torch.int32)
    s.y = torch.empty(c["rows"], c["heads"] * c["dim"], dtype=s.dt, device=DEV)
    s.turns = torch.empty(c["rot"] // 2, dtype=torch.int64, device=DEV)


def _prepare_append(s, c, seed):
    g = _gen(seed)
    s.dt = KINDS[c["dtype"]]
    s.ld, s.total = (c["hq"] + 2 * c["hk"]) * c["dim"], 4 * c["rows"] + 16
    s.x = torch.randn(c["rows"], s.ld, generator=g, device=DEV).to(s.dt)
    s.positions = torch.randint(0, c["span"], (c["rows"],), generator=g, device=DEV, dtype=torch.int32)
    s.slots = torch.randperm(s.total, generator=g, device=DEV)[:c["rows"]].to(torch.int32)
    if c["pad"]:
        s.slots[-c["pad"]:] = -1
        s.positions[-c["pad"]:] = -1
    w = c["hk"] * c["dim"]
    s.k, s.v = (torch.randn(s.total + 1, w, generator=g, device=DEV).to(s.dt) for _ in range(2))
    s.q = torch.zeros(c["rows"], c["hq"] * c["dim"], dtype=s.dt, device=DEV)
    s.turns = torch.empty(c["rot"] // 2, dtype=torch.int64, device=DEV)


def _prepare_attend(s, c, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    s.dt, P, R, per = KINDS[c["dtype"]], c["page"], c["requests"], c["per"]
    lengths = rng.permutation(_spread(R, c["lo"], c["hi"]))
    have = -(-lengths // P)
    s.pages, s.width = int(have.sum()) + 5, int(-(-c["hi"] // P))
    table = np.full((R, s.width), -1)
    table[np.arange(s.width)[None, :] < have[:, None]] = rng.permutation(s.pages)[:int(have.sum())]
    s.table = _ints(table)
    # the last `per` tokens of each request ask
    positions = np.maximum(lengths[:, None] - per + np.arange(per)[None, :], 0).reshape(-1)
    owners = np.repeat(np.arange(R), per)
    s.positions = _ints(np.concatenate([positions, np.full(c["pad"], -1)]))
    s.owners = _ints(np.concatenate([owners, np.full(c["pad"], -1)]))
    s.rows = R * per + c["pad"]
    w = c["hk"] * c["dim"]
    s.k, s.v = (torch.empty(s.pages * P, w, dtype=s.dt, device=DEV).normal_(generator=g) for _ in range(2))
    s.q = (1.5 * torch.randn(s.rows, c["hq"] * c["dim"], generator=g, device=DEV)).to(s.dt)
    s.o = torch.zeros_like(s.q)
    s.lse = torch.zeros(s.rows, c["hq"], device=DEV)


def _prepare_score(s, c, seed):
    """Logits with a few likely entries a row, as a trained model gives."""
    g = _gen(seed)
    s.dt, n, V = KINDS[c["dtype"]], c["rows"], c["vocab"]
    x = torch.randn(n, c["ld"], generator=g, device=DEV) * 2.0
    likely = torch.randint(0, V, (n, 6), generator=g, device=DEV)
    x.scatter_add_(1, likely, torch.rand(n, 6, generator=g, device=DEV) * 12.0)
    s.x = x.to(s.dt)
    pick = torch.randint(0, 6, (n, 1), generator=g, device=DEV)
    s.tokens = likely.gather(1, pick).reshape(-1).to(torch.int32)
    if n > 8:
        s.tokens[::9] = -1  # prompt tokens, not scored
    s.dlp = torch.randn(n, generator=g, device=DEV) / n
    s.dent = torch.randn(n, generator=g, device=DEV) * (0.01 / n)
    s.logprob, s.entropy = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    s.stats = torch.empty(n, 2, device=DEV)
    s.ids = torch.empty(n, c["top"], dtype=torch.int32, device=DEV)
    s.alt = torch.empty(n, c["top"], device=DEV)
    s.dx = torch.empty(n, V, dtype=s.dt, device=DEV) if c["back"] else None


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


def _own_plan(s, a):
    c = s.c
    a.add("sj_paged_plan", None, s.lengths, s.counts, c["requests"], c["page"], s.pages, s.table, s.width, s.free,
          s.free.numel(), s.head, s.after, s.starts, s.positions, s.slots, s.owners, s.rows, s.summary)
    return dict(table=s.table, starts=s.starts, positions=s.positions, slots=s.slots, owners=s.owners, after=s.after,
                summary=s.summary)


def _plain_plan(s):
    c, P, R = s.c, s.c["page"], s.c["requests"]
    n, m = s.lengths.long(), s.counts.long()
    have, want = (n + P - 1) // P, (n + m + P - 1) // P
    need = want - have
    ends = torch.cumsum(m, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    first = torch.cumsum(need, 0) - need
    head = s.head.long()[0]
    total, taken = ends[-1], need.sum()
    status = ((head + taken > s.free.numel()).long() + 2 * (want.max() > s.width).long() + 4 * (total > s.rows).long()
              + 8 * ((n < 0) | (m < 0)).any().long())
    ok = status == 0
    last = s.free.numel() - 1
    col = torch.arange(s.width, device=DEV)[None, :]
    fresh = (col >= have[:, None]) & (col < want[:, None]) & ok
    at = (head + first[:, None] + col - have[:, None]).clamp(0, last)
    table = torch.where(fresh, s.free.long()[at], s.table0.long())
    t = torch.arange(s.rows, device=DEV)
    live = (t < total) & ok
    owner = torch.searchsorted(ends, t, right=True).clamp(max=R - 1)
    pos = n[owner] + t - starts[owner]
    page = table[owner, (pos // P).clamp(0, s.width - 1)]
    good = live & (page >= 0) & (page < s.pages)
    i32 = torch.int32
    return dict(table=table.to(i32), starts=torch.where(ok, starts, 0).to(i32), positions=torch.where(live, pos, -1).to(i32),
                slots=torch.where(good, page * P + pos % P, -1).to(i32), owners=torch.where(live, owner, -1).to(i32),
                after=torch.where(ok, n + m, n).to(i32),
                summary=torch.stack([torch.where(ok, total, 0), head + torch.where(ok, taken, 0), status,
                                     (n + m).max()]).to(i32))


def _plain_frequencies(c, sc):
    """Angles per position, in 64 bits: far positions lose theirs in 32."""
    d = c["rot"]
    i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
    theta = sc["theta"]
    if sc["kind"] == BASE:
        theta = theta * sc["factor"] ** (d / (d - 2)) if d > 2 else theta
    f = theta ** (-2.0 * i / d)
    if sc["kind"] == LINEAR:
        f = f / sc["factor"]
    if sc["kind"] == PARTS:
        n = sc["context"] * f / (2.0 * math.pi)
        keep = ((n - sc["slow"]) / (sc["fast"] - sc["slow"])).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / sc["factor"])
    return f


def _plain_rotate(c, x, heads, positions, inverse):
    """x [rows][heads * dim] fp32, rotated."""
    d, D = c["rot"], c["dim"]
    angle = positions.double()[:, None] * _plain_frequencies(c, _scaling(c))[None, :]
    amp = _amplitude(c)
    cos, sin = (amp * angle.cos()).float()[:, None, :], (amp * angle.sin()).float()[:, None, :]
    if inverse:
        sin = -sin
    x = x.reshape(-1, heads, D)
    if c["layout"] == HALF:
        a, b = x[..., :d // 2], x[..., d // 2:d]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., d:]], -1).reshape(-1, heads * D)


def _own_turns(s):
    """The frequency table, made once and kept by the program."""
    from sejong_amd import _native as N
    c, sc = s.c, _scaling(s.c)
    scaling = N.RopeScaling(sc["theta"], sc["kind"], sc["factor"], sc["context"], sc["fast"], sc["slow"])
    N.api.sj_rope_frequencies(None, s.turns.data_ptr(), c["rot"], ctypes.byref(scaling))


def _own_rope(s, a):
    c = s.c
    _own_turns(s)
    a.add("sj_rope_rows", None, s.x, s.ld, s.y, c["heads"] * c["dim"], CODES[c["dtype"]], c["rows"], c["heads"],
          c["dim"], c["rot"], c["layout"], s.positions, s.turns, _amplitude(c), int(c["inverse"]))
    return s.y


def _plain_rope(s):
    c = s.c
    x = s.x[:, :c["heads"] * c["dim"]].float()
    return _plain_rotate(c, x, c["heads"], s.positions, c["inverse"]).to(s.dt)


def _own_append(s, a):
    c, size = s.c, s.x.element_size()
    _own_turns(s)
    q = s.x.data_ptr()
    k, v = q + c["hq"] * c["dim"] * size, q + (c["hq"] + c["hk"]) * c["dim"] * size
    a.add("sj_paged_append", None, q, s.ld, k, s.ld, v, s.ld, CODES[c["dtype"]], c["rows"], c["hq"], c["hk"], c["dim"],
          c["rot"], c["layout"], s.positions, s.slots, s.turns, _amplitude(c), s.q, c["hq"] * c["dim"], s.k, s.v,
          c["hk"] * c["dim"], s.total)
    return dict(q=s.q, k=s.k[:s.total], v=s.v[:s.total])


def _plain_append(s):
    c = s.c
    a, b = c["hq"] * c["dim"], (c["hq"] + c["hk"]) * c["dim"]
    x = s.x.float()
    q = _plain_rotate(c, x[:, :a], c["hq"], s.positions, False).to(s.dt)
    k = _plain_rotate(c, x[:, a:b], c["hk"], s.positions, False).to(s.dt)
    live = s.slots >= 0
    at = torch.where(live, s.slots, s.total).long()  # the row behind the last slot takes what is not kept
    s.k[at], s.v[at] = k, s.x[:, b:]
    return dict(q=torch.where(live[:, None], q, s.q), k=s.k[:s.total], v=s.v[:s.total])


def _own_attend(s, a):
    c, w = s.c, s.c["hk"] * s.c["dim"]
    need = a.lib.sj_paged_attention_workspace_bytes(s.rows, c["hq"], c["hk"], c["dim"])
    s.work = torch.empty(max(int(need), 256), dtype=torch.uint8, device=DEV)
    a.add("sj_paged_attention", None, s.q, c["hq"] * c["dim"], s.k, s.v, w, CODES[c["dtype"]], s.pages, c["page"],
          s.table, s.width, c["requests"], s.owners, s.positions, s.rows, c["hq"], c["hk"], c["dim"], c["window"], s.o,
          c["hq"] * c["dim"], s.lse, s.work, s.work.numel())
    return dict(o=s.o, lse=s.lse)


def _plain_attend(s):
    c, P, D = s.c, s.c["page"], s.c["dim"]
    n, hk, g = s.rows, c["hk"], c["hq"] // c["hk"]
    j = torch.arange(c["hi"], device=DEV)
    pos, owner = s.positions.long()[:, None], s.owners.long()
    page = s.table.long()[owner.clamp(min=0)][:, j // P]
    seen = (j[None, :] <= pos) & (page >= 0) & (page < s.pages) & (owner >= 0)[:, None]
    if c["window"]:
        seen &= j[None, :] > pos - c["window"]
    slot = torch.where(seen, page * P + j % P, 0)
    k = s.k[slot].float().view(n, -1, hk, D).permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(s.q.float().view(n, hk, g, D) * D ** -0.5, k)
    del k
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = (score - top).exp()
    total = e.sum(-1, keepdim=True)
    v = s.v[slot].float().view(n, -1, hk, D).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    live = (s.positions >= 0) & (s.owners >= 0)
    lse = (top + total.log()).reshape(n, -1)
    return dict(o=torch.where(live[:, None], o.reshape(n, -1), 0.0).to(s.dt), lse=torch.where(live[:, None], lse, 0.0))


def _own_score(s, a):
    c, n, V = s.c, s.c["rows"], s.c["vocab"]
    need = a.lib.sj_token_logprobs_workspace_bytes(n, V, c["top"])
    s.work = torch.empty(max(int(need), 256), dtype=torch.uint8, device=DEV)
    code = CODES[c["dtype"]]
    a.add("sj_token_logprobs", None, s.x, code, c["ld"], n, V, s.tokens, c["top"], s.logprob, s.entropy, s.stats, s.ids,
          s.alt, s.work, s.work.numel())
    out = dict(logprob=s.logprob, entropy=s.entropy, ids=s.ids, alternatives=s.alt)
    if c["back"]:
        a.add("sj_token_logprobs_bwd", None, s.x, code, c["ld"], n, V, s.tokens, s.stats, s.entropy, s.dlp, s.dent, s.dx,
              code, V)
        out["dx"] = s.dx
    return out


def _plain_score(s):
    c, V = s.c, s.c["vocab"]
    x = s.x[:, :V].float()
    m = x.amax(-1, keepdim=True)
    # the sum without one of its largest terms, which is 1: what a peaked row
    # holds beside its peak would be lost next to it
    rest = torch.where(x < m, (x - m).exp(), 0.0).sum(-1, keepdim=True) + ((x == m).sum(-1, keepdim=True) - 1)
    lp = x - m - rest.log1p()
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plp.sum(-1)
    scored = (s.tokens >= 0) & (s.tokens < V)
    at = s.tokens.long().clamp(0, V - 1)[:, None]
    logprob = torch.where(scored, lp.gather(1, at)[:, 0], 0.0)
    # whole keys in the order of the values, the lowest index first among equals
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    keys = order * (1 << 20) - torch.arange(V, device=DEV)
    ids = (-torch.topk(keys, c["top"], dim=-1).values) & ((1 << 20) - 1)
    out = dict(logprob=logprob, entropy=entropy, ids=ids.to(torch.int32), alternatives=lp.gather(1, ids))
    if c["back"]:
        hot = (torch.arange(V, device=DEV)[None, :] == at) & scored[:, None]
        dlp = torch.where(scored, s.dlp, 0.0)[:, None]
        dx = dlp * torch.where(hot, -lp.expm1(), -p) - s.dent[:, None] * (plp + p * entropy[:, None])
        out["dx"] = dx.to(s.dt)
    return out


# ------------------------------------------------------------------- work

def work(c):
    kind = c["kind"]
    if kind == "plan":
        R, P = c["requests"], c["page"]
        n, m = _plan_sizes(c)
        pages = int((-(-(n + m) // P) - -(-n // P)).sum())
        return dict(bytes=4 * (2 * R + 2 * R + 1 + 3 * _capacity(c) + 2 * pages + R), flops=0)
    size = 4 if c["dtype"] == "f32" else 2
    if kind == "rope":
        n = c["rows"] * c["heads"]
        return dict(bytes=2 * n * c["dim"] * size + 4 * c["rows"], flops=3 * n * c["rot"])
    if kind == "append":
        rows, heads = c["rows"] - c["pad"], c["hq"] + 2 * c["hk"]
        return dict(bytes=2 * rows * heads * c["dim"] * size + 8 * c["rows"], flops=3 * rows * (c["hq"] + c["hk"]) * c["rot"])
    if kind == "attend":
        last, per = _spread(c["requests"], c["lo"], c["hi"]), c["per"]
        window = c["window"] or 1 << 40
        # the tokens of one request read the same keys
        keys = int(np.minimum(last, window + per - 1).sum())
        seen = sum(int(np.minimum(np.maximum(last - per + 1 + i, 1), window).sum()) for i in range(per))
        rows = c["requests"] * per
        return dict(bytes=2 * keys * c["hk"] * c["dim"] * size + rows * c["hq"] * (2 * c["dim"] * size + 4),
                    flops=4 * seen * c["hq"] * c["dim"])
    n, V = c["rows"], c["vocab"]
    return dict(bytes=n * V * size * (2 if c["back"] else 1) + n * (16 + 8 * c["top"]), flops=n * V * (14 if c["back"] else 6))


# ------------------------------------------------------------------ exact

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](s, case)


def _exact_plan(s, c):
    P = c["page"]
    n, m, free = s.lengths.cpu().numpy(), s.counts.cpu().numpy(), s.free.cpu().numpy()
    table = s.table0.cpu().numpy().copy()
    out = np.full((3, s.rows), -1, np.int32)
    starts, at, head = [0], 0, 3
    for r in range(len(n)):
        for col in range(-(-int(n[r]) // P), -(-int(n[r] + m[r]) // P)):
            table[r, col] = free[head]
            head += 1
        pos = np.arange(n[r], n[r] + m[r])
        out[0, at:at + m[r]] = pos
        out[1, at:at + m[r]] = table[r, pos // P] * P + pos % P
        out[2, at:at + m[r]] = r
        at += int(m[r])
        starts.append(at)
    return dict(table=table, starts=np.array(starts, np.int32), positions=out[0], slots=out[1], owners=out[2], after=n + m,
                summary=np.array([at, head, 0, (n + m).max()], np.int32))


def _exact_turn(c, x, heads, positions, inverse):
    """Rotation as a complex product, 64 bits."""
    d, sc = c["rot"], _scaling(c)
    f = []
    for i in range(d // 2):
        theta = sc["theta"]
        if sc["kind"] == BASE and d > 2:
            theta *= math.pow(sc["factor"], d / (d - 2))
        w = math.exp(-2.0 * i / d * math.log(theta))
        if sc["kind"] == LINEAR:
            w /= sc["factor"]
        elif sc["kind"] == PARTS:
            n = sc["context"] * w / (2.0 * math.pi)
            g = min(1.0, max(0.0, (n - sc["slow"]) / (sc["fast"] - sc["slow"])))
            w = g * w + (1.0 - g) * w / sc["factor"]
        f.append(w)
    f = torch.tensor(f, dtype=torch.float64, device=DEV)
    angle = positions.double()[:, None] * f
    turn = torch.polar(torch.full_like(angle, _amplitude(c)), -angle if inverse else angle)[:, None, :]
    y = x.double().reshape(-1, heads, c["dim"]).clone()
    first = slice(0, d // 2) if c["layout"] == HALF else slice(0, d, 2)
    second = slice(d // 2, d) if c["layout"] == HALF else slice(1, d, 2)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(-1, heads * c["dim"])


def _exact_rope(s, c):
    return _exact_turn(c, s.x[:, :c["heads"] * c["dim"]], c["heads"], s.positions, c["inverse"])


def _exact_append(s, c):
    a, b = c["hq"] * c["dim"], (c["hq"] + c["hk"]) * c["dim"]
    rows = c["rows"] - c["pad"]
    q = s.q.double()
    q[:rows] = _exact_turn(c, s.x[:rows, :a], c["hq"], s.positions[:rows], False)
    k, v = s.k[:s.total].double(), s.v[:s.total].double()
    k[s.slots[:rows].long()] = _exact_turn(c, s.x[:rows, a:b], c["hk"], s.positions[:rows], False)
    v[s.slots[:rows].long()] = s.x[:rows, b:].double()
    return dict(q=q, k=k, v=v)


def _exact_attend(s, c):
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


def _exact_score(s, c):
    n, V = c["rows"], c["vocab"]
    found = dict(logprob=[], entropy=[], ids=[], alternatives=[], dx=[])
    step = max(1, (1 << 25) // V)
    for r in range(0, n, step):
        x = s.x[r:r + step, :V].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        t = s.tokens[r:r + step].long()
        scored = t >= 0
        found["logprob"].append(torch.where(scored, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0))
        h = -torch.xlogy(p, p).sum(-1)
        found["entropy"].append(h)
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        found["ids"].append(best.to(torch.int32))
        found["alternatives"].append(lp.gather(1, best))
        if c["back"]:
            dlp = torch.where(scored, s.dlp[r:r + step].double(), 0.0)[:, None]
            dx = -p * (dlp + s.dent[r:r + step].double()[:, None] * (lp + h[:, None]))
            dx.scatter_add_(1, t.clamp(min=0)[:, None], dlp)
            found["dx"].append(dx.float() if s.dt is torch.bfloat16 else dx)
    return {k: torch.cat(v) for k, v in found.items() if v}
