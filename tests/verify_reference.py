"""The rejection rule in 64 bits on the host, one sequence and one position after
the other: what verify_draft and verify_sets are compared with."""
import numpy as np

NEAR = 1e-11   # a decision this near its border says nothing (double sums of up to 2^18 terms differ by less)


def chances(x, t=1.0, words=None):
    """softmax(x / t) over the allowed ids; t <= 0 or NaN: all on the first of the
    largest. NaN and -inf are not allowed, +inf is the largest finite float.
    Zeros where nothing is allowed."""
    z = np.asarray(x, np.float64).copy()
    z[np.isnan(z)] = -np.inf
    z = np.minimum(z, np.float64(np.finfo(np.float32).max))
    if words is not None:
        bits = np.unpackbits(np.ascontiguousarray(words).view(np.uint8), bitorder="little")[: z.size]
        z[bits == 0] = -np.inf
    p = np.zeros(z.size)
    if z.max() == -np.inf:
        return p
    if not t > 0:
        p[np.argmax(z)] = 1.0
        return p
    ok = z > -np.inf
    p[ok] = np.exp((z[ok] - z.max()) / np.float64(t))
    return p / p.sum()


def dense(idx, prob, count, size):
    """A kept set as a dense vector."""
    p = np.zeros(size)
    for i, v in zip(idx[:count], prob[:count]):
        p[i] = np.float64(v) if v > 0 else 0.0
    return p


def draw(w, u):
    """The drawn id and how near u came to a border (relative to the whole)."""
    at = np.flatnonzero(w > 0)
    c = np.cumsum(w[at])
    reach = np.flatnonzero(c >= u * c[-1])
    k = int(reach[0]) if reach.size else at.size - 1
    return int(at[k]), float(np.min(np.abs(c / c[-1] - u))) if u > 0 else 1.0


def verify(p_of, q_of, draft, u_accept, u_draw):
    """One sequence: p_of(i), q_of(i) its distributions (q_of None: certain
    drafts). (tokens, acceptance probabilities, nearest border)."""
    n = len(draft)
    tokens, shares, near = [], [], 1.0
    for i in range(n + 1):
        p = p_of(i)
        w = p
        if i < n:
            d = int(draft[i])
            q = q_of(i) if q_of is not None else np.eye(1, p.size, d)[0] if 0 <= d < p.size else np.zeros(p.size)
            inside = 0 <= d < p.size
            pd, qd = (p[d], q[d]) if inside else (0.0, 0.0)
            shares.append(min(1.0, pd / qd) if qd > 0 else float(pd > 0))
            if qd > 0 and 0 < u_accept[i]:
                near = min(near, abs(u_accept[i] - pd / qd))
            if u_accept[i] * qd < pd:
                tokens.append(d)
                continue
            w = np.maximum(p - q, 0.0)
            if not w.sum() > 0:
                w = p
        if w.sum() > 0:
            t, b = draw(w, u_draw)
            near = min(near, b)
            tokens.append(t)
        break
    return tokens, shares, near
