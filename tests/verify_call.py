"""One verify_draft call on tensors as they are, checked against the rule in 64 bits:
for tests that set the logits' bits themselves."""
import numpy as np
import torch

import verify_reference as R


def to(a, dtype=None):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def bits(t):
    """A logits tensor's bits as a whole-number view."""
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


# NaN by its bits: quiet and signalling, of either sign
NANS = {torch.float32: (0x7FC00000, -0x400000, 0x7F800001, -0x7FFFFF), torch.bfloat16: (0x7FC0, -0x40, 0x7F81, -0x7F)}


def made_up(seed, B, K, V, dtype, lens=None, extra=0, near=0.5):
    """Logits of target and drafter (with `extra` rows of NaN behind each, of no sequence),
    drafts that are the drafter's samples, uniforms, lengths and first rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    lens = np.full(B, K, np.int32) if lens is None else np.asarray(lens, np.int32)
    ts = np.concatenate([[0], np.cumsum(lens + 1)[:-1]]).astype(np.int32)
    ds = np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.int32)
    rows, D = int(lens.sum()) + B, int(lens.sum())
    x = torch.full((rows + extra, V), float("nan"), dtype=dtype, device="cuda")
    y = torch.full((D + extra, V), float("nan"), dtype=dtype, device="cuda")
    z = torch.randn((rows, V), generator=g, device="cuda") * 2.5
    z.scatter_(1, torch.randint(0, V, (rows, 3), generator=g, device="cuda"), 11.0)
    at = torch.from_numpy(np.concatenate([ts[b] + np.arange(lens[b]) for b in range(B)]).astype(np.int64)).cuda()
    x[:rows] = z.to(dtype)
    y[:D] = (z[at] + torch.randn((D, V), generator=g, device="cuda") * near).to(dtype)
    noise = torch.empty((D, V), device="cuda").exponential_(generator=g).log_()
    d = np.zeros(D + extra, np.int32)
    d[:D] = (y[:D].float() - noise).argmax(1).cpu().numpy()
    return dict(x=x, y=y, d=d, u=rng.random(D + extra), v=rng.random(B), lens=lens, ts=ts, ds=ds, K=K)


def call(hs, c, t=None, td=None, drafter=True, mask=None, dmask=None, **kw):
    return hs.verify_draft(c["x"], to(c["d"]), to(c["u"]), to(c["v"]), c["K"], draft_logits=c["y"] if drafter else None,
                           temperature=to(t, np.float32), draft_temperature=to(td, np.float32), mask=to(mask, np.int32),
                           draft_mask=to(dmask, np.int32), n_draft=to(c["lens"]), target_start=to(c["ts"]),
                           draft_start=to(c["ds"]), **kw)


def check(out, c, tol, t=None, td=None, drafter=True, mask=None, dmask=None):
    """Tokens and counts equal, acceptance probabilities within `tol` of their value."""
    torch.cuda.synchronize()
    B, K = len(c["lens"]), c["K"]
    rows, drafted = int(c["ts"][-1] + c["lens"][-1]) + 1, int(c["ds"][-1] + c["lens"][-1])
    x, y = c["x"][:rows].float().cpu().numpy(), c["y"][:drafted].float().cpu().numpy()
    T = np.ones(B, np.float32) if t is None else np.asarray(t, np.float32)
    TD = np.ones(B, np.float32) if td is None else np.asarray(td, np.float32)
    tokens, count, accept = (out[k].cpu().numpy() for k in ("tokens", "count", "accept"))
    want = []
    for b in range(B):
        s0, t0, n = c["ds"][b], c["ts"][b], c["lens"][b]
        p_of = lambda i: R.chances(x[t0 + i], T[b], None if mask is None else mask[t0 + i])  # noqa: E731,B023
        q_of = (lambda i: R.chances(y[s0 + i], TD[b], None if dmask is None else dmask[s0 + i])) if drafter else None  # noqa: E731,B023
        toks, shares, near = R.verify(p_of, q_of, c["d"][s0:s0 + n], c["u"][s0:s0 + n], c["v"][b])
        assert near > R.NEAR, f"sequence {b}: the test's uniform is at a border"
        assert list(tokens[b]) == toks + [-1] * (K + 1 - len(toks)), f"sequence {b}"
        assert count[b] == len(toks), f"sequence {b}"
        full = np.array(shares + [-1.0] * (n - len(shares)))
        np.testing.assert_allclose(accept[s0:s0 + n], full, rtol=tol, atol=1e-37, err_msg=f"sequence {b}")
        want.append(toks)
    return want
