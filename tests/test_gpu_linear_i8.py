"""quantize_rows and linear_i8 against whole numbers and 64 bits on the host.

Rows in 8 bits: q is the whole number nearest to 127 x / max |x| (halves to even),
equal everywhere: in double 127 x is exact, the quotient's halves are exact, and any
other quotient of two 24-bit numbers by each other is at least 2^-33 of itself away
from a half, farther than its rounding. scale is max |x| / 127 rounded once.

The product's sum is a whole number, exact; its conversion, the two scales and the
bias are at most four roundings of 2^-24 of the magnitudes P = |sum s s| + |bias|; the
activations are evaluated to within 2^-20 of |y| and stretch an error by at most 1.13
(GELU's largest slope); the residual and the result round once more, the result by half
a step of its type."""
import ctypes

import numpy as np
import pytest

from test_gpu_linear import ACTS, act64, half_step

pytestmark = pytest.mark.gpu


def quantized(x):
    """(q, scale) of float64 rows."""
    top = np.abs(x).max(axis=-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(top > 0, np.rint(x * 127 / top), 0.0)
    return q, (top[..., 0].astype(np.float32) / np.float32(127))


def compare_rows(hs, x, **kw):
    import torch
    q, s = hs.quantize_rows(x, **kw)
    torch.cuda.synchronize()
    want_q, want_s = quantized(x.double().cpu().numpy())
    assert np.array_equal(q.cpu().numpy().astype(np.float64), want_q)
    assert np.array_equal(s.cpu().numpy(), want_s)
    return q, s


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 7), (3, 8), (2, 100), (5, 1000), (64, 4096), (33, 8192), (4, 8193), (2, 20000), (300, 65)])
@pytest.mark.parametrize("pad", [0, 3])
def test_rows(hs, M, K, pad, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(M + K)
    buf = torch.full((M, K + pad), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    x = buf[:, :K]
    x.copy_(torch.randn((M, K), generator=g, device="cuda") * torch.rand((M, 1), generator=g, device="cuda"))
    x[M // 2] = 0 if M > 2 else x[M // 2]
    full = torch.full((M, K + 5), 99, dtype=torch.int8, device="cuda")
    compare_rows(hs, x, q=full[:, :K])
    assert torch.all(full[:, K:] == 99)


def test_rows_halves_and_extremes(hs):
    """Quotients on a half, rows of the smallest and largest values."""
    import torch
    rows = []
    for top in (127.0, 254.0, 1.0, 127.0 * 2**-30, 2.0**-126, 2.0**-149, 3 * 2.0**-149, 127 * 2.0**-149, 2.0**-121, 1e-38, 3.0e38, 2.0**127):
        steps = np.arange(-127, 128, dtype=np.float64)
        x = np.concatenate([steps * top / 127, (steps + 0.5)[:-1] * top / 127, [top, -top, 0.0, top / 2, -top / 2]])
        rows.append(x.astype(np.float32))
    x = torch.from_numpy(np.stack(rows)).cuda()
    compare_rows(hs, x)
    compare_rows(hs, x.to(torch.bfloat16).nan_to_num(posinf=3e38, neginf=-3e38))


def test_rows_that_are_not_finite(hs):
    import torch
    x = torch.randn((4, 50), device="cuda")
    x[1, 3], x[2, 4], x[3, 5] = float("inf"), float("nan"), float("-inf")
    for t in (x, x.to(torch.bfloat16), x.half()):
        q, s = hs.quantize_rows(t)
        torch.cuda.synchronize()
        assert torch.isfinite(s[0]) and torch.all(torch.isnan(s[1:])) and not torch.any(q[1:])
    w = torch.ones((3, 50), dtype=torch.int8, device="cuda")
    y = hs.linear_i8(q, s, w, torch.ones(3, device="cuda"))
    torch.cuda.synchronize()
    assert torch.all(torch.isfinite(y[0])) and torch.all(torch.isnan(y[1:]))


def compare(got, x, xs, w, ws, bias, act, c, res):
    dt = got.dtype
    sums = x.double().cpu().numpy() @ np.swapaxes(w.double().cpu().numpy(), -1, -2)       # below 2^31: exact
    y = sums * xs.double().cpu().numpy()[..., :, None] * ws.double().cpu().numpy()[..., None, :]
    P = np.abs(y)
    if bias is not None:
        b = bias.double().cpu().numpy()[..., None, :]
        y, P = y + b, P + np.abs(b)
    z = act64(y, act, c)
    r = 0.0 if res is None else res.double().cpu().numpy()
    want = z + r
    tol = 1.13 * 4 * 2.0**-24 * P + (2.0**-20 * np.abs(y) if act not in ("none", "relu") else 0) + 2.0**-24 * (np.abs(z) + np.abs(r))
    tol = tol + half_step(dt) * (np.abs(want) + tol) + (2.0**-25 if "float16" in str(dt) and "bfloat" not in str(dt) else 1e-38)
    g = got.double().cpu().numpy()
    assert g.shape == want.shape
    off = np.abs(g - want) / tol
    assert np.all(np.isfinite(g)) and off.max() <= 1.0, f"{off.max()} times the bound at {np.unravel_index(off.argmax(), off.shape)}"


def tensors(seed, G, M, K, N, dtype, bias, residual, pad=0, offset=0, shared=True):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16

    def make(kind, *shape, scale=1.0):
        """Rows `pad` elements apart, `offset` elements in."""
        rows = int(np.prod(shape[:-1]))
        width = shape[-1] + pad
        if kind == torch.int8:
            buf = torch.full((offset + rows * width + 1,), 127, dtype=kind, device="cuda")
            fill = torch.randint(-128, 128, shape, generator=g, device="cuda").to(kind)
        else:
            buf = torch.full((offset + rows * width + 1,), float("nan"), dtype=kind, device="cuda")
            fill = torch.randn(shape, generator=g, device="cuda") * scale
        t = buf[offset:offset + rows * width].view(*shape[:-1], width)[..., :shape[-1]]
        t.copy_(fill)
        return t

    lead = () if G is None else (G,)
    one = G is not None and shared
    x = make(torch.int8, *(() if one else lead), M, K)
    xs = torch.rand((*(() if one else lead), M), generator=g, device="cuda") * 0.02 + 0.001
    if one:
        x, xs = x.expand(G, M, K), xs.expand(G, M)
    ws = (torch.rand((*lead, N), generator=g, device="cuda") + 0.1) * K**-0.5 * 0.02
    return (x, xs, make(torch.int8, *lead, N, K), ws, make(dt, *lead, N, scale=0.5) if bias else None,
            make(dt, *lead, M, N) if residual else None)


def one(hs, seed, G, M, K, N, dtype, act, out="same", bias=True, residual=True, pad=0, offset=0, shared=True):
    import torch
    x, xs, w, ws, b, r = tensors(seed, G, M, K, N, dtype, bias, residual, pad, offset, shared)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    full = torch.full((*w.shape[:-2], M, N + 3), 77.0, dtype=torch.float32 if out == "f32" else dt, device="cuda")
    got = hs.linear_i8(x, xs, w, ws, bias=b, act=act, act_param=3.0, residual=r, dtype=dt, out=full[..., :N])
    torch.cuda.synchronize()
    assert torch.all(full[..., N:] == 77.0)
    compare(got, x, xs, w, ws, b, act, 3.0, r)


SIZES = [
    (1, 1, 1), (1, 64, 64), (1, 4096, 4096), (1, 16, 3), (2, 100, 17), (1, 127, 33), (1, 1000, 130), (3, 896, 50), (5, 65, 1000),
    (15, 256, 256), (16, 512, 100), (17, 128, 64), (31, 4112, 48), (32, 640, 96), (33, 96, 500), (48, 2048, 257), (64, 1024, 512),
    (65, 72, 65), (100, 208, 300), (127, 333, 129), (128, 128, 128), (129, 512, 640), (256, 1024, 256), (257, 272, 513),
    (320, 512, 1111), (512, 256, 768), (700, 64, 1024), (1024, 192, 520), (1500, 400, 2000),
]


@pytest.mark.parametrize("dtype,out", [("bf16", "same"), ("f16", "f32")])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_sizes(hs, M, K, N, dtype, out):
    one(hs, M + K + N, None, M, K, N, dtype, ACTS[(M + K + N) % 6], out)


@pytest.mark.parametrize("M,K,N,G", [(200, 528, 4100, None), (256, 80, 3900, None), (64, 16, 16380, None), (60, 272, 4000, 4),
                                     (256, 2048, 4096, None), (600, 256, 9000, None), (1100, 160, 9000, None)])
def test_blocks_per_cu(hs, M, K, N, G):
    """Sizes of about one block, of two and of more tiles for each of the 256 CUs."""
    one(hs, M + K, G, M, K, N, "bf16", ACTS[(M + K) % 6], "f32")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,out", [("bf16", "same"), ("bf16", "f32"), ("f16", "same"), ("f16", "f32")])
@pytest.mark.parametrize("M,K,N,G", [(100, 80, 34_002, None), (384, 400, 16_500, None), (128, 1040, 9000, 5)])
def test_one_and_a_half_to_two_tiles_a_cu(hs, M, K, N, G, act, dtype, out):
    """Tiles of 128 x 128, two of them to a CU."""
    one(hs, M + K, G, M, K, N, dtype, act, out)


@pytest.mark.parametrize("M,K,N", [(1, 4096, 96), (7, 130, 50), (64, 513, 257), (130, 528, 300), (300, 1024, 520)])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (3, 5), (16, 0), (16, 16), (8, 8)])
def test_strides_and_alignment(hs, M, K, N, pad, offset):
    one(hs, M + K, None, M, K, N, "bf16", "silu", pad=pad, offset=offset)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,out", [("bf16", "same"), ("bf16", "f32"), ("f16", "same"), ("f16", "f32")])
@pytest.mark.parametrize("M", [1, 64, 200])
def test_epilogues(hs, M, act, dtype, out):
    for bias in (False, True):
        for residual in (False, True):
            one(hs, 5 + bias + 2 * residual, None, M, 256, 144, dtype, act, out, bias, residual)


@pytest.mark.parametrize("M,K,N,G", [(1, 512, 128, 3), (20, 200, 70, 5), (64, 256, 256, 4), (150, 96, 130, 2), (300, 320, 300, 3)])
@pytest.mark.parametrize("shared", [True, False])
def test_groups(hs, M, K, N, G, shared):
    one(hs, G, G, M, K, N, "bf16", "silu", shared=shared, pad=2)


@pytest.mark.parametrize("M", [1, 70, 300])
def test_largest_sums(hs, M):
    """131071 products of -128 by -128: 2^31 - 2^14, and of -128 by 127."""
    import torch
    K = 131071
    x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    y = hs.linear_i8(x, torch.ones(M, device="cuda"), w, torch.ones(3, device="cuda"), out_dtype=torch.float32)
    torch.cuda.synchronize()
    want = np.array([K * 16384, -K * 128 * 127, K * 16384], np.float32)
    assert np.array_equal(y.cpu().numpy(), np.tile(want, (M, 1)))
    over = hs.LinearI8Args(1, K + 1, 1, 1, hs.BF16, hs.F32)
    over.x = over.weight = x.data_ptr()
    over.x_stride = over.weight_stride = K + 1
    over.x_scale = over.weight_scale = over.out = y.data_ptr()
    assert hs.lib().ultima_hsamp_linear_i8(ctypes.byref(over), None) in (hs.ERR_UNSUPPORTED, hs.ERR_INVALID)


@pytest.mark.parametrize("M", [1, 64, 256])
def test_the_same_every_time_captured_or_not(hs, M):
    import torch

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn((M, 1024), generator=g, device="cuda").to(torch.bfloat16)
        return (x, *tensors(seed, None, M, 1024, 512, "bf16", True, True)[2:])

    state = inputs(1)

    def step(out=None, stream=None, work=(None, None)):
        x, w, ws, b, r = state
        q, s = hs.quantize_rows(x, *work, stream=stream)
        return hs.linear_i8(q, s, w, ws, bias=b, act="gelu", residual=r, out=out, stream=stream)

    out = torch.empty((M, 512), dtype=torch.bfloat16, device="cuda")
    keep = torch.empty((M, 1024), dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, work=keep)
    s = torch.cuda.Stream()
    for seed in range(5, 9):
        for t, n in zip(state, inputs(seed)):
            t.copy_(n)
        want = step()
        torch.cuda.synchronize()
        other = step(stream=s)
        out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)


def test_over_its_residual_and_heads_side_by_side(hs):
    import torch
    x, xs, w, ws, b, r = tensors(3, None, 40, 256, 320, "bf16", True, True)
    want = hs.linear_i8(x, xs, w, ws, bias=b, act="silu", residual=r)
    hs.linear_i8(x, xs, w, ws, bias=b, act="silu", residual=r, out=r)
    x, xs, w, ws, b, q = tensors(8, 4, 50, 128, 96, "bf16", True, True)
    out = torch.zeros((50, 4, 96), dtype=torch.bfloat16, device="cuda")
    got = hs.linear_i8(x, xs, w, ws, bias=b, act="silu", residual=q, out=out.transpose(0, 1))
    torch.cuda.synchronize()
    assert torch.equal(r, want)
    compare(got, x, xs, w, ws, b, "silu", 0, q)


def test_past_32_bit_offsets(hs):
    """A weight of more than 2^32 bytes: the last rows."""
    import torch
    K, N = 32768, 140000
    w = torch.zeros((N, K), dtype=torch.int8, device="cuda")
    w[-64:] = torch.randint(-127, 128, (64, K), device="cuda").to(torch.int8)
    ws = torch.full((N,), 1e-4, device="cuda")
    for M in (1, 200):
        x = torch.randint(-127, 128, (M, K), device="cuda").to(torch.int8)
        xs = torch.full((M,), 1e-3, device="cuda")
        got = hs.linear_i8(x, xs, w, ws, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert not torch.any(got[:, :-64])
        compare(got[:, -64:], x, xs, w[-64:], ws[-64:], None, "none", 0, None)
