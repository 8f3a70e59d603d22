"""verify_draft where a logit is not a number, by its bits.

NaN is not allowed whatever its bits and sign: no row emits its id, no draft of it is
accepted, and no sum has it. Acceptance probabilities as in the other tests: a double
quotient rounded to float, 2^-24 of the value, and 1e-12 for the sums behind it."""
import numpy as np
import pytest

import verify_call as C

pytestmark = pytest.mark.gpu

ACCEPT_TOL = 2.0 ** -24 + 1e-12


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("side", ["target", "drafter", "both"])
@pytest.mark.parametrize("at", [0, 8200])      # in a whole slice, in the row's last ids
def test_greedy_rows_never_take_a_nan(hs, dtype, side, at):
    """The largest logit of a greedy row is +inf, or the largest float of its type; NaN
    stands at lower ids near it. The drafts are such a NaN's id, the largest's id, others."""
    import torch
    dt = getattr(torch, dtype)
    B, K, V = 8, 2, 9001
    c = C.made_up(5, B, K, V, dt)
    for rows in ([c["x"]] if side != "drafter" else []) + ([c["y"]] if side != "target" else []):
        for k, nan in enumerate(C.NANS[dt]):
            C.bits(rows)[:, at + 3 + 130 * k] = nan
        rows[::2, at + 700] = float("inf")
        rows[1::2, at + 700] = torch.finfo(dt).max
    c["d"][:] = np.resize([at + 700, at + 3, at + 133, at + 263, at + 700, 17], B * K)
    t = [0.0 if side != "drafter" else 1.0] * B
    td = [0.0 if side != "target" else 1.0] * B
    want = C.check(C.call(hs, c, t, td), c, ACCEPT_TOL, t, td)
    if side != "drafter":
        assert all(w[-1] == at + 700 for w in want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("extra", [0, 900])      # with the rows behind the last sequence: a large call
def test_nan_of_every_kind_has_no_weight(hs, dtype, masked, extra):
    """Quiet and signalling NaN of both signs among the logits of both sides."""
    import torch
    dt = getattr(torch, dtype)
    B, K, V = 6, 4, 40001
    c = C.made_up(6, B, 200 if extra else K, V, dt, lens=[K] * B, extra=extra)
    rows, D = B * (K + 1), B * K
    g = torch.Generator(device="cuda").manual_seed(1)
    for t, n in ((c["x"], rows), (c["y"], D)):
        for r in range(n):
            for k, nan in enumerate(C.NANS[dt]):
                if r % 6 in (k, 4):              # one kind, all of them, none
                    C.bits(t)[r, torch.randint(0, V, (9,), generator=g, device="cuda")] = nan
    mask = dmask = None
    if masked:
        rng = np.random.default_rng(2)
        mask, dmask = (rng.integers(-2**31, 2**31, (n + extra, -(-V // 32)), dtype=np.int64).astype(np.int32) for n in (rows, D))
    # float sums' quotients (bf16, large): 45 2^-24 each, see the kernel
    tol = ACCEPT_TOL + (2 * 45 * 2.0 ** -24 if extra and dtype == "bfloat16" else 0.0)
    C.check(C.call(hs, c, mask=mask, dmask=dmask), c, tol, mask=mask, dmask=dmask)
