"""Plain 64-bit forms of the paged decoding operators, and a captured graph
of library calls on a stream of its own."""
import ctypes
import math

import numpy as np

from tests import gpu_util as G


def rotate(x, heads, D, rot, layout, positions, freq, amplitude=1.0, inverse=False):
    """x [rows][heads * D] float64, rotated (layout 0: pairs (2i, 2i + 1), 1: (i, i + rot / 2))."""
    y = np.array(x, np.float64).reshape(len(x), heads, D)
    angle = np.asarray(positions, np.float64)[:, None] * freq
    c, s = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None] * (-1.0 if inverse else 1.0)
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout else (slice(0, rot, 2), slice(1, rot, 2))
    ya, yb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = ya * c - yb * s, ya * s + yb * c
    return y.reshape(len(x), heads * D)


def frequencies(rot, theta=10000.0, kind=0, factor=1.0, context=0.0, fast=0.0, slow=0.0):
    f = np.zeros(rot // 2)
    for i in range(rot // 2):
        t = theta * factor ** (rot / (rot - 2.0)) if kind == 2 and rot > 2 else theta
        w = t ** (-2.0 * i / rot)
        if kind == 1:
            w /= factor
        if kind == 3:
            g = min(1.0, max(0.0, (context * w / (2 * math.pi) - slow) / (fast - slow)))
            w = w * g + w * (1 - g) / factor
        f[i] = w
    return f


def attention(q, k, v, table, P, pages, owners, positions, hq, hk, D, window=0):
    """(o, lse, tol scale sum p|v|, score error scale) in float64 of every row; None where the row is left out."""
    out = []
    for r in range(len(q)):
        if positions[r] < 0 or not 0 <= owners[r] < len(table):
            out.append(None)
            continue
        n = min(positions[r] + 1, table.shape[1] * P)
        j = np.arange(max(0, positions[r] + 1 - window) if window else 0, n)
        page = table[owners[r]][j // P]
        fine = (page >= 0) & (page < pages)
        slot = page[fine].astype(np.int64) * P + j[fine] % P
        o, lse, mag, err = np.zeros((hq, D)), np.full(hq, -np.inf), np.zeros((hq, D)), np.zeros(hq)
        for h in range(hq):
            kk, vv = k[slot][:, h // (hq // hk)], v[slot][:, h // (hq // hk)]
            qq = q[r, h]
            with np.errstate(invalid="ignore"):
                s = kk @ qq * D ** -0.5
            keep = s != -np.inf
            if not keep.any():
                continue
            s, vv, kk = s[keep], vv[keep], kk[keep]
            m = s.max()
            e = np.exp(s - m)
            o[h], lse[h] = e @ vv / e.sum(), m + np.log(e.sum())
            mag[h] = e @ np.abs(vv) / e.sum()
            err[h] = (np.abs(kk) @ np.abs(qq)).max() * D ** -0.5 * (D + 4) * 2.0 ** -24 + (len(s) + 64) * 2.0 ** -24
        out.append((o, lse, mag, err))
    return out


def plan(lengths, counts, P, pages, table, free, head, capacity):
    """The step's plan, or the status of one that cannot be."""
    table = table.copy()
    n, m = lengths.astype(np.int64), counts.astype(np.int64)
    rows = np.full((3, capacity), -1, np.int32)
    starts = np.zeros(len(n) + 1, np.int32)
    status, need, want = 0, 0, 0
    if len(n):
        good = (n >= 0) & (m >= 0)
        gn, gm = np.where(good, n, 0), np.where(good, m, 0)
        need, want = int((-(-(gn + gm) // P) - -(-gn // P)).sum()), int((-(-(gn + gm) // P)).max())
        status |= 8 * int((~good).any() or (gn + gm).max() > 2 ** 31 - 1)
        status |= 4 * int(gm.sum() > capacity)
    status |= 1 * int(head < 0 or head + need > len(free)) | 2 * int(want > table.shape[1])
    if status:
        return dict(status=status, head=head, starts=starts, rows=rows, table=table, after=lengths.copy())
    at = 0
    for r in range(len(n)):
        for c in range(-(-int(n[r]) // P), -(-int(n[r] + m[r]) // P)):
            table[r, c] = free[head]
            head += 1
        pos = np.arange(n[r], n[r] + m[r])
        page = table[r, pos // P].astype(np.int64)
        rows[0, at:at + len(pos)] = pos
        rows[1, at:at + len(pos)] = np.where((page >= 0) & (page < pages), page * P + pos % P, -1)
        rows[2, at:at + len(pos)] = r
        at += len(pos)
        starts[r + 1] = at
    return dict(status=0, head=head, starts=starts, rows=rows, table=table, after=(n + m).astype(np.int32))


class Graph:
    """Calls of `record(stream)` captured once and replayed; the runtime is the one that the library has loaded."""

    def __init__(self, record):
        from sejong_amd import _native as N
        N.load()
        self.hip = hip = ctypes.CDLL("libamdhip64.so.7")
        self.stream, graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        self.do(hip.hipStreamCreate(ctypes.byref(self.stream)))
        self.do(hip.hipStreamBeginCapture(self.stream, 2))
        record(self.stream)
        self.do(hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)))
        self.do(hip.hipGraphInstantiate(ctypes.byref(self.exe), graph, None, None, ctypes.c_size_t(0)))
        self.do(hip.hipGraphDestroy(graph))

    @staticmethod
    def do(status):
        assert status == 0, f"HIP {status}"

    def replay(self):
        self.do(self.hip.hipGraphLaunch(self.exe, self.stream))
        self.do(self.hip.hipStreamSynchronize(self.stream))

    def close(self):
        self.do(self.hip.hipGraphExecDestroy(self.exe))
        self.do(self.hip.hipStreamDestroy(self.stream))


def ints(a):
    return G.dev(np.asarray(a, np.int32), "i32")


def turns(rot, **kw):
    """The frequency table on the device."""
    from sejong_amd import _native as N
    t = G.empty(max(rot // 2, 1) * 8, "u8")
    sc = N.RopeScaling(kw.get("theta", 10000.0), kw.get("kind", 0), kw.get("factor", 1.0), kw.get("context", 0.0),
                       kw.get("fast", 0.0), kw.get("slow", 0.0))
    N.api.sj_rope_frequencies(None, t.p, rot, ctypes.byref(sc))
    return t
