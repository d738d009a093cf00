"""Plain forms of beam search's selection (64 bits) and of the pages' fork,
compaction and copy."""
import numpy as np

NO_PAGES, ROWS, LENGTHS, LIST_FULL = 1, 4, 8, 16


def select(x, scores, beams, keep, lengths=None, ended=None, end=-1, power=0.0):
    """x [rows][V] float64.  The candidates' ranks too, in their order, for tests of what lies near each other."""
    rows, V = x.shape
    lengths = np.zeros(rows, int) if lengths is None else lengths
    ended = np.zeros(rows, int) if ended is None else ended
    out = dict(parents=[], tokens=[], scores=[], lengths=[], ended=[], ranks=[])
    for g in range(rows // beams):
        found = []
        for b in range(beams):
            r = g * beams + b
            s = float(scores[r])
            if not np.isfinite(s):
                continue
            if ended[r]:
                found.append((-s / max(int(lengths[r]), 1) ** power, b * V + max(end, 0), s, r, end))
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                m = x[r].max()
                lse = m + np.log(np.exp(x[r] - m).sum())
            if not np.isfinite(lse):
                continue
            total = s + (x[r] - lse)
            f = max(int(lengths[r]) + 1, 1) ** power
            found += [(-total[v] / f, b * V + v, total[v], r, v) for v in range(V) if x[r, v] > -np.inf]
        found.sort(key=lambda c: c[:2])
        for c in found[:keep]:
            was = ended[c[3]] != 0
            for key, value in zip(out, (c[3], c[4], c[2], lengths[c[3]] + (not was), was or c[4] == end, -c[0])):
                out[key].append(value)
        for _ in range(keep - len(found[:keep])):
            for key, value in zip(out, (-1, -1, -np.inf, 0, 1, -np.inf)):
                out[key].append(value)
    return {k: np.array(v, float if k in ("scores", "ranks") else np.int32) for k, v in out.items()}


def fork(parents, table, lengths, P, pages, shared, free, head):
    """Every holder of every page counted anew; -> dict, or the status of a step that cannot be."""
    R, before = len(parents), len(lengths)
    lengths = np.asarray(lengths, np.int64)
    void = dict(table=np.full((R, table.shape[1]), -1), lengths=np.zeros(R, int), shared=shared.copy(), free=free.copy(),
                copies=np.tile([-1, -1, 0], (R, 1)), taken=0, head=head, back=0)
    status = 0
    if (np.asarray(parents) >= before).any() or (lengths < 0).any() or (-(-lengths // P) > table.shape[1]).any():
        return dict(void, status=LENGTHS | (NO_PAGES if head < 0 or head > len(free) else 0))
    out = {k: np.array(v) for k, v in void.items()}

    def fine(p):
        return 0 <= p < pages

    change, heirs, taken = np.zeros(pages, int), set(), 0
    for r in range(before):
        for p in table[r, :-(-lengths[r] // P)]:
            if fine(p):
                change[p] -= 1
    for i, r in enumerate(parents):
        if r < 0:
            continue
        n = int(lengths[r])
        row = table[r, :-(-n // P)].copy()
        if n % P and fine(row[-1]) and (r in heirs or shared[row[-1]] > 0):
            if 0 <= head + taken < len(free):
                out["copies"][i] = [row[-1], free[head + taken], n % P]
                row[-1] = -1  # its own page: counted below
            taken += 1
        heirs.add(r)
        for p in row:
            if fine(p):
                change[p] += 1
        if out["copies"][i, 0] >= 0:
            row[-1] = out["copies"][i, 1]
        out["table"][i, :len(row)], out["lengths"][i] = row, n
    if head < 0 or head + taken > len(free):
        return dict(void, status=NO_PAGES)
    out["shared"] = shared + change
    head += taken
    back = np.flatnonzero(out["shared"] < 0).tolist()
    for i, p in enumerate(back[:head]):
        out["free"][head - 1 - i], out["shared"][p] = p, 0
    given = min(len(back), head)
    return dict(out, status=LIST_FULL if given < len(back) else 0, taken=taken, head=head - given, back=given)


def compact(table, lengths, P, pages, after, shared, free, head, capacity):
    rest = [int(p) for p in free[max(head, 0):]]
    below = [p for p in rest if 0 <= p < after]
    known = set(rest)
    moves = [p for p in range(after, pages) if p not in known]
    status = NO_PAGES * (head < 0 or head > len(free) or len(moves) > len(below)) | ROWS * (len(moves) > capacity)
    copies = np.tile([-1, -1, 0], (capacity, 1))
    if status:
        return dict(status=status, table=table, shared=shared, free=free, copies=copies, moves=0, head=head, left=0)
    to = dict(zip(moves, below))
    out = np.full_like(table, -1)
    for r, n in enumerate(lengths):
        for c in range(min(-(-max(int(n), 0) // P), table.shape[1])):
            p = int(table[r, c])
            out[r, c] = to.get(p, -1 if p >= after else p) if 0 <= p < pages else -1
    s = np.where(np.arange(pages) < after, shared, 0)
    for i, p in enumerate(moves):
        s[to[p]] = shared[p]
        copies[i] = [p, to[p], P]
    left = below[len(moves):]
    f = np.full(len(free), -1)
    f[len(free) - len(left):] = left
    return dict(status=0, table=out, shared=s, free=f, copies=copies, moves=len(moves), head=len(free) - len(left),
                left=len(left))


def copy(cache, copies, P, width):
    """cache [layers][pages * P][ld], in place."""
    pages = cache.shape[1] // P
    for f, t, n in np.asarray(copies).tolist():
        if 0 <= f < pages and 0 <= t < pages and n > 0:
            cache[:, t * P:t * P + min(n, P), :width] = cache[:, f * P:f * P + min(n, P), :width]
    return cache
