"""Token log probabilities, entropy, alternatives and their gradient in 64
bits, from the definitions."""
import numpy as np


def scores(x, tokens, top=0):
    x = np.asarray(x, np.float64)
    n, V = x.shape
    m = x.max(1, keepdims=True)
    ref = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(x - ref)
    # the sum without one largest term, as a peaked row needs it
    rest = np.where(x == m, 0.0, e).sum(1, keepdims=True) + (x == m).sum(1, keepdims=True) - 1.0
    none = ~np.isfinite(m) & (m < 0)
    ll = np.where(none, 0.0, np.log1p(rest))
    lp = x - ref - ll
    p = np.where(none, 0.0, np.exp(lp))
    with np.errstate(invalid="ignore"):
        entropy = -np.where(p > 0, p * lp, 0.0).sum(1)
    tokens = np.asarray(tokens)
    ok = (tokens >= 0) & (tokens < V)
    at = np.where(ok, tokens, 0)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return dict(lp=lp, p=p, ll=ll[:, 0], ref=ref[:, 0], entropy=entropy, ids=order,
                logprob=np.where(ok, lp[np.arange(n), at], 0.0), alt=np.take_along_axis(lp, order, 1), ok=ok, at=at)


def gradient(x, tokens, dlp, dent):
    s = scores(x, tokens)
    lp, p = s["lp"], s["p"]
    hot = np.zeros_like(p)
    hot[np.arange(len(p)), s["at"]] = s["ok"]
    with np.errstate(invalid="ignore"):
        own = np.where(hot > 0, -np.expm1(lp), -p)
        ent = np.where(p > 0, p * (lp + s["entropy"][:, None]), 0.0)
    dlp = np.where(s["ok"], dlp, 0.0)[:, None] if dlp is not None else 0.0
    return dlp * own - (np.asarray(dent)[:, None] * ent if dent is not None else 0.0)
