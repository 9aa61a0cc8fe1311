"""kc_sample_dev's definition in the host's widest type."""
import math

import numpy as np

LD = np.longdouble


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, share, room): the token, its share of what is kept, and the least
    distance, relative to the sums compared, by which any decision was made."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    m = l.max()
    if m == -np.inf:
        return -1, 0.0, math.inf
    if not temperature > 0:
        return int(np.argmax(l)), 1.0, math.inf
    if m == np.inf:
        l, m = np.where(l == np.inf, 0.0, -np.inf), 0.0
    with np.errstate(all="ignore"):
        w = np.exp((l.astype(LD) - LD(m)) / LD(temperature)) if temperature < math.inf else LD(1) * (l > -np.inf)
        w = np.where(l == m, LD(1), np.where(l == -np.inf, LD(0), w))
    kept = np.lexsort((np.arange(len(l)), -l))
    if 0 < top_k < len(l):
        kept = kept[:top_k]
    room = math.inf
    if top_p < 1:
        upto = np.cumsum(w[kept])
        want = LD(top_p) * upto[-1]
        room = float(np.min(np.abs(upto - want)) / max(want, LD(1)))
        kept = kept[:1 + int(np.sum(upto[:-1] < want))]
    if min_p > 0:
        least = min(float(min_p), 1.0)
        off = np.abs(w[kept] - LD(least))
        room = min(room, float(np.min(off[off > 0], initial=np.inf)) / least)
        kept = kept[w[kept] >= LD(least)]
    kept = np.sort(kept)
    kept = kept[w[kept] > 0]
    upto = np.cumsum(w[kept])
    want = LD(min(max(u, 0.0) if u == u else 0.0, 1 - 2.0 ** -24)) * upto[-1]
    room = min(room, float(np.min(np.abs(upto - want)) / upto[-1]))
    token = int(kept[int(np.sum(upto <= want))])
    return token, float(w[token] / upto[-1]), room
