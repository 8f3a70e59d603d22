"""linear (act(x W^T + bias) + residual) against 64 bits on the host.

The sum of K exact products in float: each addition is off by at most one step of
its partial sum (2^-23, matrix instructions need not round to nearest), K of them
by K 2^-23 of the sum of magnitudes S. The activations are evaluated in float,
to within 2^-20 of |y| (their functions to a few steps of 2^-24, once or twice
through a factor up to 1), and stretch an error by at most 1.13 (GELU's largest
slope). The result's rounding: half a step of its type."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def act64(y, act, c):
    if act == "relu":
        return np.maximum(y, 0)
    if act == "silu":
        return y / (1 + np.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))
    if act == "softcap":
        return c * np.tanh(y / c)
    return y


def half_step(dt):
    import torch
    return torch.finfo(dt).eps / 2


def compare(got, x, w, bias, act, c, res, dt):
    x, w = (t.double().cpu().numpy() for t in (x, w))
    K = x.shape[-1]
    y = x @ np.swapaxes(w, -1, -2)
    S = np.abs(x) @ np.swapaxes(np.abs(w), -1, -2)
    if bias is not None:
        b = bias.double().cpu().numpy()[..., None, :]
        y, S = y + b, S + np.abs(b)
    z = act64(y, act, c)
    r = 0.0 if res is None else res.double().cpu().numpy()
    want = z + r
    tol = 1.13 * (K + 1) * 2.0**-23 * S + 2.0**-20 * np.abs(y) + 2.0**-23 * (np.abs(z) + np.abs(r))
    tol = tol + half_step(dt) * (np.abs(want) + tol) + 1e-38
    if dt is not None and "float16" in str(dt) and "bfloat" not in str(dt):
        tol = tol + 2.0**-25          # half's subnormals
    g = got.double().cpu().numpy()
    assert g.shape == want.shape
    off = np.abs(g - want) / tol
    assert np.all(np.isfinite(g)) and off.max() <= 1.0, f"{off.max()} times the bound at {np.unravel_index(off.argmax(), off.shape)}"


def tensors(seed, G, M, K, N, dtype, bias, residual, pad=0, offset=0, shared=True):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16

    def make(*shape, scale=1.0):
        """Rows `pad` elements apart, `offset` elements into NaN."""
        rows = math.prod(shape[:-1])
        buf = torch.full((offset + rows * (shape[-1] + pad) + 1,), float("nan"), dtype=dt, device="cuda")
        t = buf[offset:offset + rows * (shape[-1] + pad)].view(*shape[:-1], shape[-1] + pad)[..., :shape[-1]]
        t.copy_(torch.randn(shape, generator=g, device="cuda") * scale)
        return t

    lead = () if G is None else (G,)
    x = make(M, K) if G is None else make(M, K).expand(G, M, K) if shared else make(G, M, K)
    return (x, make(*lead, N, K, scale=K**-0.5), make(*lead, N, scale=0.5) if bias else None,
            make(*lead, M, N) if residual else None)


ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "softcap"]


def one(hs, seed, G, M, K, N, dtype, act, out="same", bias=True, residual=True, pad=0, offset=0, shared=True):
    import torch
    x, w, b, r = tensors(seed, G, M, K, N, dtype, bias, residual, pad, offset, shared)
    dt = torch.float32 if out == "f32" else x.dtype
    # rows of the output apart, what lies between them left alone
    full = torch.full((*w.shape[:-2], M, N + 3), 77.0, dtype=dt, device="cuda")
    got = hs.linear(x, w, bias=b, act=act, act_param=3.0, residual=r, out=full[..., :N])
    torch.cuda.synchronize()
    assert torch.all(full[..., N:] == 77.0)
    compare(got, x, w, b, act, 3.0, r, dt)


SIZES = [
    (1, 1, 1), (1, 64, 64), (1, 4096, 4096), (1, 8, 3), (2, 100, 17), (1, 127, 33), (1, 1000, 130),
    (3, 896, 50), (5, 65, 1000), (15, 256, 256), (16, 512, 100), (17, 64, 64), (31, 4100, 48), (32, 640, 96), (33, 96, 500),
    (48, 2048, 257), (64, 1024, 512), (65, 72, 65), (100, 200, 300), (127, 333, 129), (128, 128, 128), (129, 512, 640),
    (256, 1024, 256), (257, 264, 513), (320, 512, 1111), (512, 256, 768), (700, 64, 1024), (1024, 192, 520),
]


@pytest.mark.parametrize("dtype,out", [("bf16", "same"), ("f16", "f32")])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_sizes(hs, M, K, N, dtype, out):
    one(hs, M + K + N, None, M, K, N, dtype, ACTS[(M + K + N) % 6], out)


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "same")])
@pytest.mark.parametrize("M,K,N,G", [(200, 520, 4100, None), (256, 72, 3900, None), (129, 1000, 5400, None), (64, 8, 16380, None),
                                     (60, 264, 4000, 4), (256, 2048, 4096, None)])
def test_linear_of_a_block_per_cu(hs, M, K, N, G, dtype, out):
    """Sizes whose 64 x 64 tiles are about one for each of the 256 CUs."""
    one(hs, M + K, G, M, K, N, dtype, ACTS[(M + K) % 6], out)


@pytest.mark.parametrize("M,K,N", [(1, 4096, 96), (7, 130, 50), (64, 513, 257), (130, 520, 300), (300, 1024, 520)])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (3, 5), (8, 0), (8, 8), (4, 4)])
def test_linear_strides_and_alignment(hs, M, K, N, pad, offset):
    """Rows and tensors at any element's address; NaN around them."""
    one(hs, M + K, None, M, K, N, "bf16", "silu", pad=pad, offset=offset)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("M", [1, 64, 200])
def test_linear_epilogues(hs, M, act, dtype, out):
    for bias in (False, True):
        for residual in (False, True):
            one(hs, 5 + bias + 2 * residual, None, M, 256, 144, dtype, act, out, bias, residual)


@pytest.mark.parametrize("M,K,N,G", [(1, 512, 128, 3), (20, 200, 70, 5), (64, 256, 256, 4), (150, 96, 130, 2), (300, 320, 300, 3)])
@pytest.mark.parametrize("shared", [True, False])
def test_linear_groups(hs, M, K, N, G, shared):
    one(hs, G, G, M, K, N, "bf16", "silu", shared=shared, pad=2)


@pytest.mark.parametrize("M", [1, 50, 140])
def test_linear_groups_side_by_side(hs, M):
    """Four heads' outputs in one row each."""
    import torch
    x, w, b, r = tensors(8, 4, M, 128, 96, "bf16", True, True)
    out = torch.zeros((M, 4, 96), dtype=torch.bfloat16, device="cuda")
    got = hs.linear(x, w, bias=b, act="silu", residual=r, out=out.transpose(0, 1))
    torch.cuda.synchronize()
    compare(got, x, w, b, "silu", 0, r, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_over_its_residual(hs, M):
    import torch
    x, w, b, r = tensors(3, None, M, 256, 320, "bf16", True, True)
    want = hs.linear(x, w, bias=b, act="silu", residual=r)
    hs.linear(x, w, bias=b, act="silu", residual=r, out=r)
    torch.cuda.synchronize()
    assert torch.equal(r, want)


@pytest.mark.parametrize("M", [1, 64, 256])
def test_linear_is_the_same_every_time_captured_or_not(hs, M):
    import torch
    x, w, b, r = tensors(4, None, M, 1024, 512, "bf16", True, True)
    out = torch.empty((M, 512), dtype=torch.bfloat16, device="cuda")
    hs.linear(x, w, bias=b, act="gelu", residual=r, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hs.linear(x, w, bias=b, act="gelu", residual=r, out=out)
    s = torch.cuda.Stream()
    for seed in range(5, 9):
        for t, n in zip((x, w, b, r), tensors(seed, None, M, 1024, 512, "bf16", True, True)):
            t.copy_(n)
        want = hs.linear(x, w, bias=b, act="gelu", residual=r)
        torch.cuda.synchronize()
        other = hs.linear(x, w, bias=b, act="gelu", residual=r, stream=s)
        out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)


@pytest.mark.parametrize("M", [1, 33, 256])
def test_linear_infinities_and_nan_stay_in_their_row(hs, M):
    """A NaN or an infinity in a row of x or W reaches that row or column alone."""
    import torch
    x, w, b, r = tensors(6, None, M, 256, 300, "bf16", True, False)
    want = hs.linear(x, w, bias=b)
    x[M // 2, 17] = float("nan")
    w[123, 200] = float("inf")
    got = hs.linear(x, w, bias=b)
    torch.cuda.synchronize()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[M // 2] = True
    hit[:, 123] = True
    assert torch.all(torch.isnan(got[M // 2])) and not torch.any(torch.isfinite(got[:, 123]))
    assert torch.equal(got[~hit], want[~hit])


def test_linear_past_32_bit_offsets(hs):
    """Weights of more than 2^32 bytes: the last rows, at offsets past 2^31 elements."""
    import torch
    K, N = 16384, 140000                  # 2.29e9 elements
    w = torch.zeros((N, K), dtype=torch.bfloat16, device="cuda")
    w[-64:] = torch.randn((64, K), device="cuda").to(torch.bfloat16) * K**-0.5
    for M in (1, 200):
        x = torch.randn((M, K), device="cuda").to(torch.bfloat16)
        got = hs.linear(x, w, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert not torch.any(got[:, :-64])
        compare(got[:, -64:], x, w[-64:], None, "none", 0, None, torch.float32)


def test_draft_heads_to_verified_tokens(hs, sampler, wl):
    """The operators as a drafter with heads uses them: two heads' residual blocks
    in one call, their logits in another, tokens and sets from the sampler, the
    target's logits, then verification; against the same steps in 64 bits from the
    logits on (the logits themselves against their bound)."""
    import torch

    import verify_reference as R
    B, K, H, V = 5, 2, 256, 1003
    g = torch.Generator(device="cuda").manual_seed(9)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)

    hidden, w1, b1, w2 = normal(B, H), normal(K, H, H, scale=H**-0.5), normal(K, H, scale=0.1), normal(V, H, scale=0.15)
    xs = hidden.expand(K, B, H)
    h = hs.linear(xs, w1, bias=b1, act="silu", residual=xs.contiguous())
    compare(h, xs, w1, b1, "silu", 0, xs, torch.bfloat16)
    y = hs.linear(h.view(K * B, H), w2, act="softcap", act_param=20.0, out_dtype=torch.float32)
    compare(y, h.view(K * B, H), w2, None, "softcap", 20.0, None, torch.float32)
    y = y.view(K, B, V).transpose(0, 1).reshape(B * K, V).contiguous()          # sequence by sequence
    rng = np.random.default_rng(10)
    to = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    drafts = sampler.run(y, [wl.identity_params(temperature=0.9)] * (B * K), to(rng.random(B * K)))["token"]
    x = hs.linear(normal(B * (K + 1), H), w2, act="softcap", act_param=20.0, out_dtype=torch.float32)
    u, v = rng.random(B * K), rng.random(B)
    u[::2] *= 0.05
    t = torch.full((B,), 0.9, device="cuda")
    out = hs.verify_draft(x, drafts, to(u), to(v), K, draft_logits=y, temperature=t, draft_temperature=t)
    torch.cuda.synchronize()
    tokens, count, d = out["tokens"].cpu().numpy(), out["count"].cpu().numpy(), drafts.cpu().numpy()
    xv, yv, tv = x.cpu().numpy(), y.cpu().numpy(), np.float32(0.9)
    for b in range(B):
        want, _, near = R.verify(lambda i: R.chances(xv[b * 3 + i], tv), lambda i: R.chances(yv[b * 2 + i], tv),
                                 d[2 * b:2 * b + 2], u[2 * b:2 * b + 2], v[b])
        assert near > R.NEAR and list(tokens[b][:count[b]]) == want


def exact_act(y, act, c):
    """Without cancellation: relative to the value itself."""
    if act == "gelu":
        return 0.5 * y * np.vectorize(math.erfc)(-y / math.sqrt(2))
    if act == "gelu_tanh":
        return y / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))
    if act == "silu":
        return y / (1 + np.exp(-y))
    return c * np.tanh(y / c)


def one_column(hs, values, act, c=0.0):
    """The activation of each value: rows of one element by a weight of one."""
    import torch
    x = values.to(torch.bfloat16).reshape(-1, 1)
    got = hs.linear(x, torch.ones((1, 1), dtype=torch.bfloat16, device="cuda"), act=act, act_param=c, out_dtype=torch.float32)
    torch.cuda.synchronize()
    return x[:, 0].double().cpu().numpy(), got[:, 0].double().cpu().numpy()


@pytest.mark.parametrize("c", [1e-45, 1e-42, 2.0**-128, 2.0**-126, 1e-30, 0.5, 1e30, 2.0**126, 2.0**127, 3.402823466e38])
def test_linear_caps_of_any_size(hs, c):
    """c tanh(y / c) for caps from the smallest float to the largest; the quotient, the
    function and the product round a few times each, and subnormal results by half of
    2^-149 (c below 2^-126: c's own steps)."""
    import torch
    c = float(np.float32(c))
    m = torch.logspace(-37, 38, 151, device="cuda")
    y, got = one_column(hs, torch.cat([torch.zeros(2, device="cuda"), -torch.zeros(1, device="cuda"), m, -m]), "softcap", c)
    with np.errstate(over="ignore"):
        want = exact_act(y, "softcap", c)
    assert np.all(np.abs(got - want) <= 16 * 2.0**-24 * np.abs(want) + 2.0**-149)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_linear_tails_of_the_activations(hs, act):
    """Each activation relative to its own value, far into the negative tail. The argument
    a of exp (erfc: its square) has at most eight roundings of its own, so that the value
    moves by 8 |a| 2^-24; twenty steps more for the functions and the products."""
    import torch
    y, got = one_column(hs, torch.linspace(-9.0, 9.0, 721, device="cuda"), act)
    want = exact_act(y, act, 0.0)
    a = {"silu": np.abs(y), "gelu": y * y, "gelu_tanh": np.abs(1.6 * y + 0.0715 * y**3)}[act]
    assert np.all(np.abs(got - want) <= (8 * a + 20) * 2.0**-24 * np.abs(want) + 1e-37)


def test_streams_of_another_device_are_refused(hs):
    import types

    import torch
    other = types.SimpleNamespace(device=torch.device("cuda", torch.cuda.current_device() + 1))
    x, w, _, _ = tensors(1, None, 2, 64, 64, "bf16", False, False)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    f64 = lambda n: torch.zeros(n, dtype=torch.float64, device="cuda")  # noqa: E731
    p = torch.zeros((2, 8), device="cuda")
    for call in (lambda: hs.linear(x, w, stream=other), lambda: hs.verify_draft(p, i32(1), f64(1), f64(1), 1, stream=other),
                 lambda: hs.verify_sets(i32(2, 8), p, i32(2), i32(1), f64(1), f64(1), 1, stream=other)):
        with pytest.raises(hs.HsampError) as e:
            call()
        assert e.value.status == hs.ERR_INVALID


def test_tensors_of_calls_on_another_stream_are_kept(hs):
    """What a call on another stream reads and writes is dropped while that stream waits;
    memory handed out meanwhile and overwritten is not theirs."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    V, B, K = 20011, 3, 2

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    x, w = normal(64, 512).to(torch.bfloat16), normal(700, 512).to(torch.bfloat16)
    b, r = normal(700).to(torch.bfloat16), normal(64, 700).to(torch.bfloat16)
    p, q = normal(B * (K + 1), V), normal(B * K, V)
    u, v = torch.rand(B * K, generator=g, device="cuda", dtype=torch.float64), torch.rand(B, generator=g, device="cuda", dtype=torch.float64)
    d, t = q.argmax(1).to(torch.int32), torch.full((B,), 0.8, device="cuda")
    n = torch.full((B,), K, dtype=torch.int32, device="cuda")
    idx = torch.arange(64, dtype=torch.int32, device="cuda").expand(B * (K + 1), 64).contiguous()
    prob, count = torch.softmax(normal(B * (K + 1), 64), 1), torch.full((B * (K + 1),), 64, dtype=torch.int32, device="cuda")
    few = d % 64
    calls = [
        (hs.linear, (x, w), dict(bias=b, residual=r)),
        (hs.verify_draft, (p, d, u, v, K), dict(draft_logits=q, temperature=t, draft_temperature=t, n_draft=n)),
        (hs.verify_sets, (idx, prob, count, few, u, v, K), dict(draft_idx=idx[:B * K].contiguous(), draft_prob=prob[:B * K].contiguous(),
                                                              draft_count=count[:B * K].contiguous(), n_draft=n)),
    ]
    s = torch.cuda.Stream()
    copy = lambda a: a.clone() if torch.is_tensor(a) else a  # noqa: E731
    for fn, args, kw in calls:
        want = fn(*args, **kw)
        mine, named = [copy(a) for a in args], {k: copy(a) for k, a in kw.items()}
        sizes = [(a.shape, a.dtype) for a in [*mine, *named.values()] if torch.is_tensor(a)]
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(100_000_000)
        got = fn(*mine, **named, stream=s)
        mine.clear()
        named.clear()
        later = [torch.full(shape, 3, dtype=dtype, device="cuda") for shape, dtype in sizes]
        torch.cuda.synchronize()
        del later
        for a, e in zip(got.values() if isinstance(got, dict) else [got], want.values() if isinstance(want, dict) else [want]):
            assert torch.equal(a, e)


def test_draft_heads_side_by_side_to_verified_sets(hs, sampler, wl):
    """Several slots, four heads each, written side by side so that the drafter's rows stand
    slot by slot as the verification takes them: each slot's tokens are the rule's on its
    own sets, whatever the other slots hold."""
    import torch

    import verify_reference as R
    B, K, H, V, cap = 5, 4, 256, 1003, 32
    g = torch.Generator(device="cuda").manual_seed(19)
    rng = np.random.default_rng(19)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)

    hidden, w, bias, lm = normal(B, H), normal(K, H, H, scale=H**-0.5), normal(K, H, scale=0.1), normal(V, H, scale=0.2)
    heads = torch.empty((B, K, H), dtype=hidden.dtype, device="cuda")
    hs.linear(hidden.expand(K, -1, -1), w, bias, act="silu", residual=hidden.expand(K, -1, -1), out=heads.transpose(0, 1))
    drafter = hs.linear(heads.view(-1, H), lm, out_dtype=torch.float32)
    h64 = hidden.double().cpu().numpy()
    y = np.einsum("bh,koh->bko", h64, w.double().cpu().numpy()) + bias.double().cpu().numpy()
    want_heads = torch.from_numpy(y / (1 + np.exp(-y)) + h64[:, None]).cuda()
    # half a step of bf16; sums of 257 terms whose magnitudes add up to less than 25 by 257 2^-23
    # of that, stretched by 1.13 at most: 9e-4
    assert torch.all((heads.double() - want_heads).abs() <= 2.0**-8 * want_heads.abs() + 1e-3)
    to = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    knobs = wl.identity_params(temperature=0.9, top_k=20)
    drafted = sampler.run(drafter, [knobs] * (B * K), to(rng.random(B * K)), want_sets=True, set_cap=cap)
    # the target's hidden states near the heads', so that drafts are accepted now and then
    state = torch.cat([heads + 0.2 * normal(B, K, H), normal(B, 1, H)], 1)
    logits = hs.linear(state.view(-1, H), lm, out_dtype=torch.float32)
    target = sampler.run(logits, [knobs] * (B * (K + 1)), to(rng.random(B * (K + 1))), want_sets=True, set_cap=cap)
    u, v = rng.random(B * K), rng.random(B)
    out = hs.verify_sets(target["kept_idx"], target["kept_prob"], target["kept_count"], drafted["token"], to(u), to(v), K,
                         draft_idx=drafted["kept_idx"], draft_prob=drafted["kept_prob"], draft_count=drafted["kept_count"])
    torch.cuda.synchronize()
    P, Q = ([r[k].cpu().numpy() for k in ("kept_idx", "kept_prob", "kept_count")] for r in (target, drafted))
    d, tokens, count = drafted["token"].cpu().numpy(), out["tokens"].cpu().numpy(), out["count"].cpu().numpy()
    for b in range(B):
        sl = slice(b * K, b * K + K)
        want, _, near = R.verify(lambda i: R.dense(*(a[b * (K + 1) + i] for a in P), V),
                                 lambda i: R.dense(*(a[b * K + i] for a in Q), V), d[sl], u[sl], v[b])
        assert near > R.NEAR and count[b] == len(want) and list(tokens[b][:len(want)]) == want
    assert any(c > 1 for c in count)
