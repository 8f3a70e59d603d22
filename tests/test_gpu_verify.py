"""verify_draft and verify_sets (verification of drafted tokens by the rejection
rule) against the rule in 64 bits on the host.

Tokens and counts are equal: every decision is made in double on both sides, and
the tests' uniforms stay 1e-11 away from the borders (checked). The acceptance
probability is one double quotient rounded to float: half a step, 2^-24 of the
value, and 1e-12 for the sums behind it. Large calls in bfloat16 (128 MB of logits at
four drafts and more, as many as their shape allows) take the sums of its rows from float exponentials: each is off by at most 3e-6 of it
(3 steps of 2^-24 of the exponent, whose mean over the weights is at most ln V < 17
by the entropy's bound: 51 2^-24; exp2's own step 2^-23; nine float additions, 9 2^-24;
62 2^-24 = 3.7e-6 in all), their quotient by twice that."""
import numpy as np
import pytest

import verify_reference as R

pytestmark = pytest.mark.gpu

ACCEPT_TOL = 2.0 ** -24 + 1e-12
ACCEPT_TOL_LARGE = 2.0 ** -24 + 2 * 62 * 2.0 ** -24
LARGE = 128 << 20


def _torch():
    import torch
    return torch, torch.device("cuda:0")


def logits(rng, rows, V, peaks=3):
    x = rng.normal(0, 2.5, (rows, V)).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, V, min(peaks, V))] = rng.normal(11, 2, min(peaks, V))
    return x


def place(x, dtype, pad=0, offset=0):
    """x on the GPU with rows `pad` elements apart and the first `offset` elements
    into its allocation, in the type; and the values it holds."""
    torch, dev = _torch()
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    rows, V = x.shape
    buf = torch.full((offset + rows * (V + pad) + 1,), float("nan"), dtype=dt, device=dev)   # between the rows: nothing to read
    t = buf[offset:offset + rows * (V + pad)].view(rows, V + pad)[:, :V]
    t.copy_(torch.from_numpy(x))
    return t, t.float().cpu().numpy()


def check(out, want, B, K, n, ds, draft_rows, tol=ACCEPT_TOL):
    tokens, count = out["tokens"].cpu().numpy(), out["count"].cpu().numpy()
    got_a = out["accept"].cpu().numpy()
    for b in range(B):
        toks, shares, near = want[b]
        assert near > R.NEAR, f"sequence {b}: the test's uniform is at a border"
        assert list(tokens[b]) == toks + [-1] * (K + 1 - len(toks)), f"sequence {b}"
        assert count[b] == len(toks), f"sequence {b}"
        full = np.array(shares + [-1.0] * (n[b] - len(shares)))
        np.testing.assert_allclose(got_a[ds[b]:ds[b] + n[b]], full, rtol=tol, atol=1e-37)


def run_draft(hs, seed, B, K, V, dtype="f32", drafter=True, n=None, t=None, td=None, mask=None, dmask=None, pad=0,
              offset=0, edit=None, near=0.5, big=False):
    """One call on made-up logits; edit(x, y, d, u, v) may change them first."""
    torch, dev = _torch()
    rng = np.random.default_rng(seed)
    lens = np.full(B, K, np.int32) if n is None else np.asarray(n, np.int32)
    ts = np.concatenate([[0], np.cumsum(lens + 1)[:-1]]).astype(np.int32)
    ds = np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.int32)
    R_, D = int(lens.sum()) + B, int(lens.sum())
    x = logits(rng, R_, V)
    at = np.concatenate([ts[b] + np.arange(lens[b]) for b in range(B)]).astype(int) if D else np.zeros(0, int)
    y = x[at] + rng.normal(0, near, (D, V)).astype(np.float32)
    d = np.array([rng.choice(V, p=R.chances(row, 0.7)) for row in y], np.int32).reshape(D)
    u, v = rng.random(D), rng.random(B)
    if edit is not None:
        edit(x, y, d, u, v)
    xt, xv = place(x, dtype, pad, offset)
    yt, yv = place(y, dtype, pad, offset) if D else (torch.empty((0, V), dtype=xt.dtype, device=dev), y)
    to = lambda a, dt: None if a is None else torch.from_numpy(np.ascontiguousarray(a, dt)).to(dev)  # noqa: E731
    out = hs.verify_draft(xt, to(d, np.int32), to(u, np.float64), to(v, np.float64), K,
                          draft_logits=yt if drafter else None, temperature=to(t, np.float32),
                          draft_temperature=to(td, np.float32), mask=None if mask is None else to(mask, np.int32),
                          draft_mask=None if dmask is None else to(dmask, np.int32),
                          n_draft=None if n is None else to(lens, np.int32),
                          target_start=None if n is None else to(ts, np.int32),
                          draft_start=None if n is None else to(ds, np.int32))
    torch.cuda.synchronize()
    T = np.ones(B, np.float32) if t is None else np.asarray(t, np.float32)
    TD = np.ones(B, np.float32) if td is None else np.asarray(td, np.float32)
    want = []
    for b in range(B):
        p_of = lambda i: R.chances(xv[ts[b] + i], T[b], None if mask is None else mask[ts[b] + i])  # noqa: E731,B023
        q_of = (lambda i: R.chances(yv[ds[b] + i], TD[b], None if dmask is None else dmask[ds[b] + i])) if drafter else None  # noqa: E731,B023
        sl = slice(ds[b], ds[b] + lens[b])
        want.append(R.verify(p_of, q_of, d[sl], u[sl], v[b]))
    large = dtype == "bf16" and K >= 4 and (B * (K + 1) + (B * K if drafter else 0)) * V * 2 > LARGE
    assert large == big, "the test is meant for the other size"
    check(out, want, B, K, lens, ds, D, ACCEPT_TOL_LARGE if large else ACCEPT_TOL)
    return want


def words_of(allowed):
    rows, V = allowed.shape
    bits = np.zeros((rows, -(-V // 32) * 32), np.uint8)
    bits[:, :V] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,K,V,pad,offset", [
    (1, 0, 1, 0, 0),              # one id, nothing drafted
    (3, 1, 1, 0, 0),
    (2, 2, 2, 1, 1),
    (5, 3, 33, 0, 1),             # rows at odd addresses, less than a load at the end
    (2, 4, 8191, 0, 0),           # one id less than a slice
    (2, 4, 8192, 8, 0),
    (2, 4, 8193, 3, 3),           # a slice of one id
    (3, 7, 50257, 0, 0),
    (1, 9, 151936, 0, 0),
    (4, 5, 16385, 0, 5),
    (70, 2, 1000, 0, 0),          # more sequences than a wave
    (1, 70, 257, 0, 0),           # more drafts than a wave
    (1, 300, 64, 0, 0),           # more drafts than a block
])
def test_draft_matches_the_rule(hs, B, K, V, pad, offset, dtype):
    run_draft(hs, 100 * B + 10 * K + V, B, K, V, dtype, pad=pad, offset=offset)


def test_draft_over_a_large_vocabulary(hs):
    """More slices than a wave: the slices' sums are scanned in pieces."""
    run_draft(hs, 3, 2, 1, 600011, "bf16")


@pytest.mark.parametrize("drafter", [True, False])
def test_draft_large_calls(hs, drafter):
    """Float exponentials first (few of the many drafts there could be): every kind
    of temperature, odd rows."""
    B = 40
    n = [i % 6 for i in range(B)]
    t = np.resize([1.0, 0.0, 0.6, 1e-38, np.inf, 3.0, np.nan, 0.8, 0.05], B)
    td = np.resize([0.8, 1.0, 0.0, 1.0], B)
    run_draft(hs, 13, B, 50 if drafter else 90, 40001, "bf16", drafter=drafter, n=n, t=t, td=td, pad=3, offset=1, big=True)


@pytest.mark.parametrize("dtype,B,K,V,big", [("bf16", 40, 50, 40001, True), ("bf16", 20, 5, 9001, False), ("f32", 20, 5, 9001, False)])
def test_draft_shifted_logits(hs, dtype, B, K, V, big):
    """Rows all below zero, rows with one slice above it, rows so far from zero that the
    product with 1 / T no longer fits the float exponentials, rows of zeroes of both
    signs."""
    n = [1 + i % 5 for i in range(B)]
    t = np.resize([1.0, 0.7, 0.0, 0.004, 2.0], B)

    def edit(x, y, d, u, v):
        for rows in (x, y):
            for r in range(rows.shape[0]):
                kind = r % 7
                if kind == 0:
                    rows[r] = -np.abs(rows[r]) - 0.5
                elif kind == 1:
                    rows[r] -= 60.0
                elif kind == 2:
                    rows[r] = -np.abs(rows[r]) - 0.5
                    rows[r, V // 2] = 3.0
                elif kind == 3:
                    rows[r] += 20000.0
                elif kind == 4:
                    rows[r] = np.where(rows[r] > 0, 0.0, -0.0)
                elif kind == 5:
                    rows[r] -= 20000.0

    run_draft(hs, 77, B, K, V, dtype, n=n, t=t, td=t, edit=edit, big=big)


def test_draft_large_calls_with_masks(hs):
    B, K, V = 24, 3, 40003
    rng = np.random.default_rng(14)
    ok = rng.random((B * (K + 1), V)) < 0.2
    okd = rng.random((B * K, V)) < 0.5
    ok[4] = False
    ok[8:12] = False
    ok[8:12, V - 1] = True
    okd[9] = False

    def edit(x, y, d, u, v):
        for a, m in ((x, ok), (y, okd)):
            r, c = np.nonzero(~m)
            a[r, c] = np.resize([np.nan, np.inf, -np.inf, np.finfo(np.float32).min], r.size)
        for i in range(B * K):
            row = ok[i // K * (K + 1) + i % K]
            d[i] = np.flatnonzero(row)[0] if row.any() else 7
        x[20, 5:9] = np.nan
        x[21, 5:9] = -np.inf
        u[::4] = 0.0
    want = run_draft(hs, 15, B, 80, V, "bf16", n=[K] * B, mask=words_of(ok), dmask=words_of(okd), edit=edit, big=True,
                     t=np.full(B, 0.8))
    assert len(want[1][0]) == 0


def test_draft_large_calls_near_the_border(hs):
    """u within 1e-5 of p / q on either side: the float sums cannot tell, and the rows
    are summed again in double."""
    import torch
    B, K, V = 24, 4, 30001

    def edit(x, y, d, u, v):
        for a in (x, y):
            a[:] = torch.from_numpy(a).to(torch.bfloat16).float().numpy()
        for b in range(B):
            for i in range(K):
                r, s = b * (K + 1) + i, b * K + i
                x[r] = y[s]
                x[r, d[s]] -= 0.5        # p / q below 1
                x[r] = torch.from_numpy(x[r]).to(torch.bfloat16).float().numpy()
                a = R.chances(x[r])[d[s]] / R.chances(y[s])[d[s]]
                u[s] = a * (1 + (3e-9 if (b + i) % 3 == 0 else -3e-9))
    want = run_draft(hs, 16, B, 100, V, "bf16", n=[K] * B, edit=edit, big=True)
    assert {len(w[0]) for w in want} == {1, 2, 3}


@pytest.mark.parametrize("drafter", [True, False])
def test_draft_ragged(hs, drafter):
    n = [0, 3, 5, 1, 0, 5, 2]
    want = run_draft(hs, 11, 7, 5, 9001, "bf16", drafter=drafter, n=n, td=[0.7] * 7)
    assert len({len(w[0]) for w in want}) > 1
    run_draft(hs, 12, 3, 4, 500, n=[0, 0, 0])


@pytest.mark.parametrize("drafter", [True, False])
def test_draft_temperatures(hs, drafter):
    """Greedy on either side, both, cold, hot, and infinite (every id alike)."""
    t = [0.0, -1.0, 1.0, 0.0, 0.05, 30.0, np.inf, 1e-38, np.nan, 0.6]
    td = [1.0, 0.7, 0.0, 0.0, 0.3, 30.0, 1.0, 1.0, 0.0, -2.0]
    run_draft(hs, 21, 10, 4, 3001, drafter=drafter, t=t, td=td, near=0.1)


def test_draft_greedy_ties_take_the_lowest_id(hs):
    def edit(x, y, d, u, v):
        x[:, [77, 9000, 20000]] = 20.0
        d[:] = [77, 77, 9000]
    want = run_draft(hs, 22, 1, 3, 20011, t=[0.0], edit=edit, drafter=False)
    assert want[0][0] == [77, 77, 77]


def test_draft_equal_rows_accept_everything(hs):
    def edit(x, y, d, u, v):
        y[:] = x[[0, 1, 2, 4, 5, 6]]
        u[:] = 1 - 1e-9
    want = run_draft(hs, 23, 2, 3, 5000, edit=edit)
    assert all(len(w[0]) == 4 for w in want)


def test_draft_outside_the_vocabulary_is_rejected(hs):
    """Equal rows, then the residual is empty: the token is drawn from p."""
    def edit(x, y, d, u, v):
        y[:] = x[[0, 1, 3, 4]]
        d[0], d[2] = -1, 5000
        d[3] = 2**31 - 1
    want = run_draft(hs, 24, 2, 2, 5000, edit=edit)
    assert [len(w[0]) for w in want] == [1, 1]


@pytest.mark.parametrize("u,v", [(0.0, 0.0), (1 - 2.0**-53, 1 - 2.0**-53), (0.0, 1 - 2.0**-53)])
def test_draft_uniforms_at_the_ends(hs, u, v):
    """u = 0 accepts whatever p allows; v = 0 draws the lowest id, v just below 1
    the last id that matters (compared by the sums of the two sides alone: the
    reference's last id or a later one of weight below 1e-12)."""
    torch, dev = _torch()
    rng = np.random.default_rng(25)
    x = logits(rng, 3, 9000)
    y = logits(rng, 2, 9000)
    d = np.array([5, 6], np.int32)
    to = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    out = hs.verify_draft(to(x), to(d), to(np.full(2, u)), to(np.full(1, v)), 2, draft_logits=to(y))
    got = out["tokens"].cpu().numpy()[0]
    p, q = [R.chances(r) for r in x], [R.chances(r) for r in y]
    m = next((i for i in range(2) if not u * q[i][d[i]] < p[i][d[i]]), 2)
    assert u > 0.0 or m == 2
    assert out["count"].item() == m + 1 and list(got[:m]) == list(d[:m])
    w = p[2] if m == 2 else np.maximum(p[m] - q[m], 0)
    t = got[m]
    if v == 0.0:
        assert t == np.flatnonzero(w > 0)[0]
    else:
        assert w[t] > 0 and w[t + 1:].sum() <= 1e-12 * w.sum()


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_draft_masks(hs, dtype, drafter):
    """Masked places hold NaN, infinities and the type's lowest value; some rows
    allow one id, some none (the sequence then has no token there)."""
    B, K, V = 6, 3, 9001
    rng = np.random.default_rng(31)
    ok = rng.random((B * (K + 1), V)) < 0.2
    okd = rng.random((B * K, V)) < 0.5
    ok[1 * 4:2 * 4] = False
    ok[1 * 4:2 * 4, 8999] = True          # sequence 1: one id allowed everywhere
    ok[2 * 4] = False                     # sequence 2: nothing from the start
    ok[3 * 4 + 3] = False                 # sequence 3: nothing at the end
    okd[4 * 3] = False                    # sequence 4: the drafter's row allows nothing

    def edit(x, y, d, u, v):
        for a, m in ((x, ok), (y, okd)):
            r, c = np.nonzero(~m)
            a[r, c] = np.resize([np.nan, np.inf, -np.inf, np.finfo(np.float32).min], r.size)
        for i in range(B * K):
            b = i // K
            d[i] = np.flatnonzero(ok[b * 4 + i % K])[0] if ok[b * 4 + i % K].any() else 7
        d[1 * 3:1 * 3 + 3] = 8999
        u[3 * 3:4 * 3] = 0.0              # sequence 3 accepts its drafts
    want = run_draft(hs, 32, B, K, V, dtype, drafter=drafter, mask=words_of(ok), dmask=words_of(okd) if drafter else None,
                     edit=edit, pad=5)
    assert len(want[2][0]) == 0 and len(want[3][0]) == 3


def test_draft_strange_logits(hs):
    """Not masked: +inf counts as the largest float, NaN and -inf as not allowed,
    a row of the type's lowest value is uniform over it."""
    def edit(x, y, d, u, v):
        x[0, [100, 4000]] = np.inf
        x[3, :] = -np.inf
        x[3, [3, 9, 4700]] = np.finfo(np.float32).min
        x[6, :] = np.nan
        x[6, 4999] = -80.0
        x[9, :] = -np.inf
        y[0, 50] = np.inf
        y[2, ::2] = np.nan
        y[2, 1::2] = -np.inf
        d[0], d[2], d[4] = 100, 9, 4999
    want = run_draft(hs, 33, 4, 2, 5000, edit=edit)
    assert len(want[3][0]) == 0


def test_draft_bad_rows_emit_nothing(hs):
    """Lengths and rows outside the arrays: count 0, every token -1, the other
    sequences as ever, nothing written for them."""
    torch, dev = _torch()
    rng = np.random.default_rng(41)
    V, K = 300, 3
    x, y = logits(rng, 8, V), logits(rng, 6, V)
    d = rng.integers(0, V, 6).astype(np.int32)
    n = np.array([3, -1, 4, 3, 2, 3, 0, 2**31 - 1], np.int32)
    ts = np.array([0, 0, 0, 5, -1, 4, 8, 0], np.int32)
    ds = np.array([0, 0, 0, 4, 0, 3, 0, 2**31 - 1], np.int32)
    to = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    u, v = rng.random(6), rng.random(8)
    out = {"accept": torch.full((6,), 9.0, device=dev)}
    hs.verify_draft(to(x), to(d), to(u), to(v), K, draft_logits=to(y), n_draft=to(n), target_start=to(ts),
                    draft_start=to(ds), outputs=out)
    tokens, count = out["tokens"].cpu().numpy(), out["count"].cpu().numpy()
    for b in (1, 2, 3, 4, 6, 7):
        assert count[b] == 0 and (tokens[b] == -1).all()
    for b in (0, 5):
        w, _, near = R.verify(lambda i: R.chances(x[ts[b] + i]), lambda i: R.chances(y[ds[b] + i]),
                              d[ds[b]:ds[b] + 3], u[ds[b]:ds[b] + 3], v[b])
        assert near > R.NEAR and list(tokens[b][:count[b]]) == w
    only = {"accept": torch.full((6,), 9.0, device=dev)}
    hs.verify_draft(to(x), to(d), to(u), to(v[:1]), K, draft_logits=to(y), n_draft=to(np.array([2], np.int32)),
                    target_start=to(np.array([1], np.int32)), draft_start=to(np.array([1], np.int32)), outputs=only)
    left = only["accept"].cpu().numpy()
    assert (left[[0, 3, 4, 5]] == 9.0).all() and (left[1:3] != 9.0).all()


def test_draft_keeps_the_targets_distribution(hs):
    """The first token over a grid of (drafted token, u, v), the drafts weighted
    by q: the target's p to the grid's step (each of the two uniforms is off by at
    most one step of 1/48 in every id's share)."""
    torch, dev = _torch()
    V, G = 5, 48
    rng = np.random.default_rng(51)
    x, y = rng.normal(0, 1, (2, V)).astype(np.float32), rng.normal(0, 1, (1, V)).astype(np.float32)
    d, i, j = np.meshgrid(np.arange(V), np.arange(G), np.arange(G), indexing="ij")
    B = d.size
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    out = hs.verify_draft(to(np.tile(x, (B, 1))), to(d.reshape(-1).astype(np.int32)), to((i.reshape(-1) + 0.5) / G),
                          to((j.reshape(-1) + 0.5) / G), 1, draft_logits=to(np.tile(y, (B, 1))))
    first = out["tokens"][:, 0].cpu().numpy()
    p, q = R.chances(x[0]), R.chances(y[0])
    share = np.array([np.sum(q[d.reshape(-1)][first == t]) / (G * G) for t in range(V)])
    np.testing.assert_allclose(share, p, atol=2.0 / G)


def test_draft_captured_and_on_another_stream(hs):
    """A captured call replayed with new contents each time, its workspace full of
    NaN before; two streams with workspaces of their own; every result the eager
    one's."""
    torch, dev = _torch()
    rng = np.random.default_rng(61)
    B, K, V = 3, 4, 20011
    need = hs.lib().ultima_hsamp_verify_draft_work_bytes(B, K, V)

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn((B * (K + 1), V), generator=g, device=dev) * 3
        y = x.view(B, K + 1, V)[:, :K].reshape(B * K, V) + torch.randn((B * K, V), generator=g, device=dev) * 0.5
        return [x, y.argmax(1).to(torch.int32), torch.rand(B * K, generator=g, device=dev, dtype=torch.float64),
                torch.rand(B, generator=g, device=dev, dtype=torch.float64), y]

    def call(i, **kw):
        return hs.verify_draft(*i[:4], K, draft_logits=i[4], **kw)

    held = inputs(0)
    work = torch.full((need,), 255, dtype=torch.uint8, device=dev)
    out = {}
    call(held, work=work, outputs=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held, work=work, outputs=out)
    for seed in range(1, 6):
        new = inputs(seed)
        want = call(new)
        for h, t in zip(held, new):
            h.copy_(t)
        work.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (seed, k)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    sets = [inputs(20), inputs(21)]
    want = [call(i) for i in sets]
    torch.cuda.synchronize()
    got = [call(i, stream=s, work=torch.empty(need, dtype=torch.uint8, device=dev)) for i, s in zip(sets * 4, streams * 4)]
    torch.cuda.synchronize()
    for k, o in enumerate(got):
        for name in o:
            assert torch.equal(o[name], want[k % 2][name])
    del rng


# ---- kept sets ----------------------------------------------------------------------

def make_sets(rng, rows, cap, V, counts=None):
    idx = np.full((rows, cap), -7, np.int32)
    prob = np.full((rows, cap), np.nan, np.float32)      # past the count: nothing to read
    count = rng.integers(1, min(cap, V) + 1, rows).astype(np.int32) if counts is None else np.asarray(counts, np.int32)
    for r in range(rows):
        c = count[r]
        idx[r, :c] = np.sort(rng.choice(V, c, replace=False))
        p = rng.exponential(1, c) ** 3
        prob[r, :c] = (p / p.sum()) if c else 0
    return idx, prob, count


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("B,K,cap,V", [
    (1, 0, 1, 5), (2, 1, 1, 3), (3, 4, 64, 70), (5, 3, 65, 500), (2, 8, 1024, 1100), (1, 2, 5000, 6000),
    (70, 2, 40, 50), (1, 70, 40, 60), (1, 300, 20, 30), (2, 1, 40000, 50000),
])
def test_sets_match_the_rule(hs, B, K, cap, V, drafter):
    torch, dev = _torch()
    rng = np.random.default_rng(B * 100 + K + cap)
    ragged = B > 2
    n = rng.integers(0, K + 1, B).astype(np.int32) if ragged else np.full(B, K, np.int32)
    ts = np.concatenate([[0], np.cumsum(n + 1)[:-1]]).astype(np.int32)
    ds = np.concatenate([[0], np.cumsum(n)[:-1]]).astype(np.int32)
    D = int(n.sum())
    P = make_sets(rng, D + B, cap, V)
    Q = make_sets(rng, D, cap, V)
    if D:
        # near the target's, so that drafts are accepted now and then
        for b in range(B):
            for i in range(n[b]):
                if rng.random() < 0.6:
                    for a, c in zip(Q, P):
                        a[ds[b] + i] = c[ts[b] + i]
    d = np.array([Q[0][r, rng.integers(0, Q[2][r])] for r in range(D)], np.int32).reshape(D)
    u, v = rng.random(D), rng.random(B)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    kw = dict(draft_idx=to(Q[0]), draft_prob=to(Q[1]), draft_count=to(Q[2])) if drafter else {}
    if ragged:
        kw.update(n_draft=to(n), target_start=to(ts), draft_start=to(ds))
    out = hs.verify_sets(to(P[0]), to(P[1]), to(P[2]), to(d), to(u), to(v), K, **kw)
    torch.cuda.synchronize()
    want = []
    for b in range(B):
        p_of = lambda i: R.dense(*(a[ts[b] + i] for a in P), V)  # noqa: E731,B023
        q_of = (lambda i: R.dense(*(a[ds[b] + i] for a in Q), V)) if drafter else None  # noqa: E731,B023
        sl = slice(ds[b], ds[b] + n[b])
        want.append(R.verify(p_of, q_of, d[sl], u[sl], v[b]))
    check(out, want, B, K, n, ds, D)


@pytest.mark.parametrize("B,cap", [(300, 9000), (600, 9000), (2, 70000)])
def test_sets_of_several_tiles(hs, B, cap):
    """Sets of 0 to cap ids whose tiles go to several blocks of a sequence or to one;
    the workspace holds anything. Every third sequence's drafter has the target's set
    and a draft outside it: the weights are then the target's."""
    torch, dev = _torch()
    rng = np.random.default_rng(B + cap)
    K, V = 1, cap + 500
    counts = np.minimum(cap, (rng.random(2 * B) ** 3 * (cap + 1)).astype(np.int32))
    counts[:2] = cap
    P = make_sets(rng, 2 * B, cap, V, counts)
    Q = make_sets(rng, B, cap, V, np.minimum(cap, (rng.random(B) ** 2 * (cap + 1)).astype(np.int32)))
    d = rng.integers(0, V, B).astype(np.int32)
    for b in range(B):
        if b % 3 == 0:
            for q, t in zip(Q, P):
                q[b] = t[2 * b]
            d[b] = np.setdiff1d(np.arange(V), Q[0][b, :Q[2][b]])[0]
        elif Q[2][b]:
            d[b] = Q[0][b, rng.integers(0, Q[2][b])]
    u, v = rng.random(B), rng.random(B)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    need = hs.lib().ultima_hsamp_verify_sets_work_bytes(B, cap)
    args = [to(t) for t in (*P, d, u, v)] + [K]
    kw = dict(draft_idx=to(Q[0]), draft_prob=to(Q[1]), draft_count=to(Q[2]))
    out = hs.verify_sets(*args, **kw, work=torch.full((need,), 255, dtype=torch.uint8, device=dev))
    torch.cuda.synchronize()
    want = [R.verify(lambda i: R.dense(*(a[2 * b + i] for a in P), V), lambda i: R.dense(*(a[b] for a in Q), V),  # noqa: B023
                     d[b:b + 1], u[b:b + 1], v[b]) for b in range(B)]
    check(out, want, B, K, [1] * B, np.arange(B), B)
    with pytest.raises(hs.HsampError):
        hs.verify_sets(*args, **kw, work=torch.empty(need - 1, dtype=torch.uint8, device=dev))


@pytest.mark.parametrize("cap,draft_cap,V", [(64, 60000, 61000), (60000, 64, 61000), (3, 200000, 250000), (4097, 4096, 9000),
                                             (9000, 50001, 50001)])
def test_sets_of_different_capacities(hs, cap, draft_cap, V):
    """A target's few ids among many of the drafter's, and the other way round."""
    torch, dev = _torch()
    rng = np.random.default_rng(cap + draft_cap)
    B, K = 12, 1
    P = make_sets(rng, 2 * B, cap, V, [max(1, cap - r % 3) for r in range(2 * B)])
    Q = make_sets(rng, B, draft_cap, V, [max(1, draft_cap - r % 5) for r in range(B)])
    for b in range(B):
        few, many = (P, Q) if cap < draft_cap else (Q, P)
        rf, rm = (2 * b, b) if few is P else (b, 2 * b)
        if b % 2:             # the few among the many, some of them likelier
            ids = np.sort(rng.choice(many[0][rm, :many[2][rm]], few[2][rf], replace=False))
            few[0][rf, :few[2][rf]] = ids
            at = np.searchsorted(many[0][rm, :many[2][rm]], ids)
            many[1][rm, at] = few[1][rf, :few[2][rf]] * rng.choice([0.5, 1.0, 2.0], ids.size).astype(np.float32)
    d = np.array([Q[0][r, rng.integers(0, Q[2][r])] for r in range(B)], np.int32)
    u, v = rng.random(B) * 0.5 + 0.5, rng.random(B)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    out = hs.verify_sets(*[to(t) for t in (*P, d, u, v)], K, draft_idx=to(Q[0]), draft_prob=to(Q[1]), draft_count=to(Q[2]))
    torch.cuda.synchronize()
    want = [R.verify(lambda i: R.dense(*(a[2 * b + i] for a in P), V), lambda i: R.dense(*(a[b] for a in Q), V),  # noqa: B023
                     d[b:b + 1], u[b:b + 1], v[b]) for b in range(B)]
    check(out, want, B, K, [1] * B, np.arange(B), B)
    assert any(len(w[0]) == 1 for w in want)


def test_sets_of_several_tiles_captured(hs):
    """Replays of a captured call with new contents give the eager call's tokens."""
    torch, dev = _torch()
    B, K, cap, V = 5, 3, 12000, 20000
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731

    def inputs(seed):
        rng = np.random.default_rng(seed)
        P, Q = make_sets(rng, B * (K + 1), cap, V), make_sets(rng, B * K, cap, V)
        d = np.array([Q[0][r, rng.integers(0, Q[2][r])] for r in range(B * K)], np.int32)
        return [to(t) for t in (*P, d, rng.random(B * K), rng.random(B), *Q)]

    def call(i, out):
        return hs.verify_sets(*i[:6], K, draft_idx=i[6], draft_prob=i[7], draft_count=i[8], outputs=out)

    held, out = inputs(0), {}
    call(held, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held, out)
    for seed in range(1, 5):
        new = inputs(seed)
        want = call(new, {})
        for h, t in zip(held, new):
            h.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (seed, k)


def test_sets_that_are_no_sets(hs):
    """Counts outside the capacity and rows outside the arrays: count 0 and -1
    everywhere; an empty target set: no token; an empty drafter's set: q = 0; NaN
    and negative probabilities count as 0."""
    torch, dev = _torch()
    rng = np.random.default_rng(71)
    cap, V, K = 16, 40, 1
    P = make_sets(rng, 16, cap, V, [8] * 16)
    Q = make_sets(rng, 8, cap, V, [8] * 8)
    P[2][0] = 17                       # sequence 0: cut off
    P[2][3] = -1                       # sequence 1, its last row
    Q[2][2] = 17                       # sequence 2, the drafter's
    P[2][6] = 0                        # sequence 3: empty target set
    P[2][9] = 0                        # sequence 4: empty at the end
    Q[2][5] = 0                        # sequence 5: empty drafter's set
    P[1][12, :4] = [np.nan, -1.0, -0.0, np.nan]
    d = np.array([Q[0][r, 0] for r in range(8)], np.int32)
    d[4] = P[0][8, 2]
    d[5] = P[0][10, 1]
    d[6] = P[0][12, 1]
    u, v = rng.random(8), rng.random(8)
    u[4] = 0.0
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    out = hs.verify_sets(to(P[0]), to(P[1]), to(P[2]), to(d), to(u), to(v), K, draft_idx=to(Q[0]), draft_prob=to(Q[1]),
                         draft_count=to(Q[2]))
    tokens, count = out["tokens"].cpu().numpy(), out["count"].cpu().numpy()
    for b in (0, 1, 2):
        assert count[b] == 0 and (tokens[b] == -1).all()
    for b in range(3, 8):
        w, _, near = R.verify(lambda i: R.dense(*(a[2 * b + i] for a in P), V), lambda i: R.dense(*(a[b] for a in Q), V),
                              d[b:b + 1], u[b:b + 1], v[b])
        assert near > R.NEAR
        assert count[b] == len(w) and list(tokens[b][:len(w)]) == w and (tokens[b][len(w):] == -1).all(), b
    assert count[3] == 0 and count[4] == 1


def test_sets_from_the_sampler(hs, sampler, wl):
    """Drafting, scoring and verifying with the sampler's own sets: the drafter's
    tokens and sets from run(), the target's sets from run(), then verify_sets;
    against the rule on those sets. A dense verification with the same logits and
    no cut agrees with verify_sets over whole-vocabulary sets up to what float
    probabilities can move a border."""
    torch, dev = _torch()
    rng = np.random.default_rng(81)
    B, K, V, cap = 6, 4, 5003, 64
    x = torch.from_numpy(logits(rng, B * (K + 1), V, peaks=6)).to(dev)
    rows = torch.tensor([b * (K + 1) + i for b in range(B) for i in range(K)], device=dev)
    y = x[rows] + 0.7 * torch.from_numpy(rng.normal(0, 1, (B * K, V)).astype(np.float32)).to(dev)
    knobs = wl.identity_params(temperature=0.8, top_k=40, top_p=0.95)
    ud = torch.from_numpy(rng.random(B * K)).to(dev)
    dr = sampler.run(y, [knobs] * (B * K), ud, want_sets=True, set_cap=cap)
    tg = sampler.run(x, [knobs] * (B * (K + 1)), torch.from_numpy(rng.random(B * (K + 1))).to(dev), want_sets=True,
                     set_cap=cap)
    u, v = rng.random(B * K), rng.random(B)
    out = hs.verify_sets(tg["kept_idx"], tg["kept_prob"], tg["kept_count"], dr["token"],
                         torch.from_numpy(u).to(dev), torch.from_numpy(v).to(dev), K, draft_idx=dr["kept_idx"],
                         draft_prob=dr["kept_prob"], draft_count=dr["kept_count"])
    torch.cuda.synchronize()
    P = [tg[k].cpu().numpy() for k in ("kept_idx", "kept_prob", "kept_count")]
    Q = [dr[k].cpu().numpy() for k in ("kept_idx", "kept_prob", "kept_count")]
    d = dr["token"].cpu().numpy()
    want = []
    for b in range(B):
        sl = slice(b * K, b * K + K)
        want.append(R.verify(lambda i: R.dense(*(a[b * (K + 1) + i] for a in P), V),
                             lambda i: R.dense(*(a[b * K + i] for a in Q), V), d[sl], u[sl], v[b]))
    check(out, want, B, K, [K] * B, [b * K for b in range(B)], B * K)
    assert any(len(w[0]) > 1 for w in want)


def test_large_draft_and_sets_captured(hs):
    """A large bfloat16 call (float exponentials, then double) and a call on sets in one
    graph, replayed with new contents and eager work between; every replay the
    eager calls' results."""
    torch, dev = _torch()
    B, K, V, cap = 16, 6, 40009, 200
    pitch = 64                        # many drafts could be: the call counts as large

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = torch.randint(0, K + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        ts = (torch.arange(B, device=dev) * (K + 1)).to(torch.int32)
        ds = (torch.arange(B, device=dev) * K).to(torch.int32)
        x = (torch.randn((B * (K + 1), V), generator=g, device=dev) * 3).to(torch.bfloat16)
        y = (x.view(B, K + 1, V)[:, :K].reshape(B * K, V).float() + torch.randn((B * K, V), generator=g, device=dev) * 0.5).to(torch.bfloat16)
        d = y.argmax(1).to(torch.int32)
        u = torch.rand(B * K, generator=g, device=dev, dtype=torch.float64)
        v = torch.rand(B, generator=g, device=dev, dtype=torch.float64)

        def top(z):
            p, i = torch.topk(torch.softmax(z.float(), 1), cap, dim=1)
            i, order = torch.sort(i, dim=1)
            return [i.to(torch.int32), p.gather(1, order).contiguous(),
                    torch.full((z.shape[0],), cap, dtype=torch.int32, device=dev)]
        return [x, d, u, v, y, n, ts, ds] + top(x) + top(y)

    def call(i, out=({}, {}), work=None):
        a = hs.verify_draft(*i[:4], pitch, draft_logits=i[4], n_draft=i[5], target_start=i[6], draft_start=i[7],
                            outputs=out[0], work=work)
        b = hs.verify_sets(*i[8:11], *i[1:4], pitch, draft_idx=i[11], draft_prob=i[12], draft_count=i[13], n_draft=i[5],
                           target_start=i[6], draft_start=i[7], outputs=out[1])
        return a, b

    assert B * (2 * pitch + 1) * V * 2 > LARGE
    held = inputs(0)
    work = torch.full((hs.lib().ultima_hsamp_verify_draft_work_bytes(B, pitch, V),), 255, dtype=torch.uint8, device=dev)
    accept = [torch.zeros(B * K, device=dev) for _ in range(2)]
    out = ({"accept": accept[0]}, {"accept": accept[1]})
    call(held, out, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held, out, work)
    for seed in range(1, 5):
        new = inputs(seed)
        want = call(new, ({"accept": torch.zeros(B * K, device=dev)}, {"accept": torch.zeros(B * K, device=dev)}))
        for h, t in zip(held, new):
            h.copy_(t)
        for a in accept:
            a.zero_()
        work.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            for k in w:
                assert torch.equal(o[k], w[k]), (seed, k)


def test_draft_sequences_that_share_rows(hs):
    """Two sequences on the same target rows with uniforms of their own (two samples
    of one continuation): each as if alone."""
    torch, dev = _torch()
    rng = np.random.default_rng(91)
    V, K = 7001, 2
    x, y = logits(rng, 3, V), logits(rng, 4, V)
    d = rng.integers(0, V, 4).astype(np.int32)
    u, v = rng.random(4) * 1e-3, rng.random(2)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    out = hs.verify_draft(to(x), to(d), to(u), to(v), K, draft_logits=to(y), target_start=to(np.zeros(2, np.int32)),
                          draft_start=to(np.array([0, 2], np.int32)))
    tokens, count = out["tokens"].cpu().numpy(), out["count"].cpu().numpy()
    for b in range(2):
        w, _, near = R.verify(lambda i: R.chances(x[i]), lambda i: R.chances(y[2 * b + i]), d[2 * b:2 * b + 2],
                              u[2 * b:2 * b + 2], v[b])
        assert near > R.NEAR and list(tokens[b][:count[b]]) == w


@pytest.mark.parametrize("cap", [16, 5000])
def test_sets_that_were_cut_off_leave_no_acceptance(hs, cap):
    """A set above its capacity or a count below 0 on either side: -1 for all of the
    sequence's drafts, the others' as ever, rows of no sequence as they were."""
    torch, dev = _torch()
    rng = np.random.default_rng(72)
    B, K, V = 5, 3, 6000
    n = np.array([3, 2, 3, 3, 1], np.int32)
    ts = np.concatenate([[0], np.cumsum(n + 1)[:-1]]).astype(np.int32)
    ds = np.concatenate([[0], np.cumsum(n)[:-1]]).astype(np.int32)
    D = int(n.sum())
    P, Q = make_sets(rng, D + B, cap, V, [cap] * (D + B)), make_sets(rng, D, cap, V, [cap - 3] * D)
    P[2][ts[0] + 3] = cap + 1          # sequence 0, its last row
    Q[2][ds[1]] = cap + 7              # sequence 1, the drafter's
    P[2][ts[3] + 1] = -1               # sequence 3
    d = np.array([Q[0][r, 0] for r in range(D)], np.int32)
    u, v = rng.random(D), rng.random(B)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    more = lambda a, fill: to(np.concatenate([a, np.full((2, *a.shape[1:]), fill, a.dtype)]))  # noqa: E731
    out = {"accept": torch.full((D + 2,), 9.0, device=dev)}
    hs.verify_sets(*[to(a) for a in P], more(d, 0), more(u, 0), to(v), K, draft_idx=more(Q[0], 0), draft_prob=more(Q[1], 0),
                   draft_count=more(Q[2], 0), n_draft=to(n), target_start=to(ts), draft_start=to(ds), outputs=out)
    torch.cuda.synchronize()
    accept, count = out["accept"].cpu().numpy(), out["count"].cpu().numpy()
    for b in (0, 1, 3):
        assert count[b] == 0 and (accept[ds[b]:ds[b] + n[b]] == -1.0).all()
    for b in (2, 4):
        toks, shares, near = R.verify(lambda i: R.dense(*(a[ts[b] + i] for a in P), V), lambda i: R.dense(*(a[ds[b] + i] for a in Q), V),
                                      d[ds[b]:ds[b] + n[b]], u[ds[b]:ds[b] + n[b]], v[b])
        assert near > R.NEAR and count[b] == len(toks)
        np.testing.assert_allclose(accept[ds[b]:ds[b] + n[b]], shares + [-1.0] * (n[b] - len(shares)), rtol=ACCEPT_TOL, atol=1e-37)
    assert (accept[D:] == 9.0).all()
