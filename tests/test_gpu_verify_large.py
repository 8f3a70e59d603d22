"""verify_draft's large bfloat16 calls, whose rows are summed by float exponentials first:
more than 1 GB of logits that the arrays hold, four drafts or more for each sequence.
Here most of those rows belong to no sequence (and are NaN), so that the rule in 64 bits
on the host is quick.

Tokens and counts are equal. A row's sum is off by at most 45 2^-24 of it: two roundings
of the exponent (17 2^-24 each: the mean over the weights of its magnitude is at most ln V
< 17 by the entropy's bound), exp2's own step 2^-23, nine float additions 9 2^-24. An
acceptance probability, a quotient of two such sums, by twice that and its own rounding."""
import numpy as np
import pytest

import verify_call as C
import verify_reference as R

pytestmark = pytest.mark.gpu

ACCEPT_TOL = 2.0 ** -24 + 1e-12
ACCEPT_TOL_LARGE = ACCEPT_TOL + 2 * 45 * 2.0 ** -24
LARGE = 1 << 30
V, K_MAX = 40001, 1000


def large(seed, B, lens, drafter=True):
    import torch
    extra = 6800 if drafter else 13600
    c = C.made_up(seed, B, K_MAX, V, torch.bfloat16, lens=lens, extra=extra)
    there = min(B * (K_MAX * (2 if drafter else 1) + 1), c["x"].shape[0] + (c["y"].shape[0] if drafter else 0))
    assert there * V * 2 > LARGE and c["d"].size >= 4 * B
    return c


def test_few_drafts_of_many(hs):
    """A large max_draft alone changes nothing: as exact as any small call."""
    import torch
    B = 40
    c = C.made_up(13, B, K_MAX, V, torch.bfloat16, lens=[i % 6 for i in range(B)])
    assert B * (2 * K_MAX + 1) * V * 2 > LARGE > (c["x"].shape[0] + c["y"].shape[0]) * V * 2
    C.check(C.call(hs, c), c, ACCEPT_TOL)


def test_a_quarter_of_a_gigabyte_is_not_large(hs):
    """Where doubles alone are the quicker ones, too: as exact as any small call."""
    import torch
    B = 20
    c = C.made_up(14, B, K_MAX, V, torch.bfloat16, lens=[4 + i % 3 for i in range(B)], extra=1600)
    assert LARGE > (c["x"].shape[0] + c["y"].shape[0]) * V * 2 > LARGE / 4 and c["d"].size >= 4 * B
    C.check(C.call(hs, c), c, ACCEPT_TOL)


@pytest.mark.parametrize("drafter", [True, False])
def test_temperatures(hs, drafter):
    B = 18
    t = np.resize([1.0, 0.0, 0.6, 1e-38, np.inf, 3.0, np.nan, 0.8, 0.05], B)
    td = np.resize([0.8, 1.0, 0.0, 1.0], B)
    c = large(13, B, [i % 6 for i in range(B)], drafter)
    C.check(C.call(hs, c, t, td, drafter), c, ACCEPT_TOL_LARGE, t, td, drafter)


def test_shifted_logits(hs):
    """Rows all below zero, rows with one slice above it, rows far from zero, rows of
    zeroes of both signs."""
    import torch
    B = 20
    t = np.resize([1.0, 0.7, 0.0, 0.004, 2.0], B)
    c = large(77, B, [1 + i % 5 for i in range(B)])
    for rows in (c["x"], c["y"]):
        n = rows.shape[0] - 6800
        for r in range(n):
            kind, z = r % 7, rows[r].float()
            z = {0: -z.abs() - 0.5, 1: z - 60.0, 2: -z.abs() - 0.5, 3: z + 20000.0, 4: torch.where(z > 0, 0.0, -0.0),
                 5: z - 20000.0, 6: z}[kind]
            if kind == 2:
                z[V // 2] = 3.0
            rows[r] = z.to(torch.bfloat16)
    C.check(C.call(hs, c, t, t), c, ACCEPT_TOL_LARGE, t, t)


def test_masks(hs):
    """Masked places hold NaN, infinities and the lowest value; a row that allows nothing,
    a sequence that allows one id."""
    import torch
    B, K = 12, 3
    c = large(15, B, [K] * B)
    rng = np.random.default_rng(14)
    ok, okd = np.zeros((c["x"].shape[0], V), bool), np.zeros((c["y"].shape[0], V), bool)
    ok[:B * (K + 1)], okd[:B * K] = rng.random((B * (K + 1), V)) < 0.2, rng.random((B * K, V)) < 0.5
    ok[4] = False
    ok[8:12] = False
    ok[8:12, V - 1] = True
    okd[9] = False
    for rows, m in ((c["x"][:B * (K + 1)], ok[:B * (K + 1)]), (c["y"][:B * K], okd[:B * K])):
        gone = torch.from_numpy(~m).cuda()
        strange = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min], device="cuda")
        rows[:] = torch.where(gone, strange[torch.arange(V, device="cuda") % 4].to(rows.dtype), rows)
    for i in range(B * K):
        row = ok[i // K * (K + 1) + i % K]
        c["d"][i] = np.flatnonzero(row)[0] if row.any() else 7
    c["x"][20, 5:9] = float("nan")
    c["x"][21, 5:9] = -float("inf")
    c["u"][:B * K:4] = 0.0

    def words(allowed):
        b = np.zeros((allowed.shape[0], -(-V // 32) * 32), np.uint8)
        b[:, :V] = allowed
        return np.packbits(b, axis=1, bitorder="little").view(np.int32)

    t = np.full(B, 0.8)
    mask, dmask = words(ok), words(okd)
    want = C.check(C.call(hs, c, t, mask=mask, dmask=dmask), c, ACCEPT_TOL_LARGE, t, mask=mask, dmask=dmask)
    assert len(want[1]) == 0


def test_uniforms_near_the_border(hs):
    """u within 1e-5 of p / q on either side: the float sums cannot tell, and the rows are
    summed again in double, which then gives the probability to its rounding."""
    import torch
    B, K = 24, 4
    c = large(16, B, [K] * B)
    for b in range(B):
        for i in range(K):
            r, s, d = b * (K + 1) + i, b * K + i, int(c["d"][b * K + i])
            c["x"][r] = c["y"][s]
            c["x"][r, d] = (c["y"][s, d].float() - 0.5).to(torch.bfloat16)        # p / q below 1
    x, y = c["x"][:B * (K + 1)].float().cpu().numpy(), c["y"][:B * K].float().cpu().numpy()
    for b in range(B):
        for i in range(K):
            r, s = b * (K + 1) + i, b * K + i
            a = R.chances(x[r])[c["d"][s]] / R.chances(y[s])[c["d"][s]]
            c["u"][s] = a * (1 + (3e-9 if (b + i) % 3 == 0 else -3e-9))
    want = C.check(C.call(hs, c), c, ACCEPT_TOL)
    assert {len(w) for w in want} == {1, 2, 3}


def test_captured(hs):
    """Replays with new contents and eager work between are the eager calls' results."""
    import torch
    B = 8
    held = large(1, B, [5] * B)
    gpu = {k: C.to(held[k]) for k in ("d", "u", "v", "lens", "ts", "ds")}

    def call(c, **kw):
        return hs.verify_draft(c["x"], c["d"], c["u"], c["v"], K_MAX, draft_logits=c["y"], n_draft=c["lens"],
                               target_start=c["ts"], draft_start=c["ds"], **kw)

    fixed = dict(held, **gpu)
    work = torch.empty(hs.lib().ultima_hsamp_verify_draft_work_bytes(B, K_MAX, V), dtype=torch.uint8, device="cuda")
    out = {}
    call(fixed, outputs=out, work=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(fixed, outputs=out, work=work)
    for seed in range(2, 6):
        new = large(seed, B, [5] * B)
        for k in ("d", "u", "v"):
            gpu[k].copy_(C.to(new[k]))
        held["x"].copy_(new["x"])
        held["y"].copy_(new["y"])
        want = call(fixed)
        work.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out["tokens"], want["tokens"]) and torch.equal(out["count"], want["count"]), seed
        assert torch.equal(out["accept"][:5 * B], want["accept"][:5 * B]), seed
