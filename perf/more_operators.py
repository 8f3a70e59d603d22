"""The operators around the vocabulary's matrix, as timed cases.

Five calls of a program that serves draft heads and trains them on what it serves:

  i8       hsamp.quantize_rows + hsamp.linear_i8: act(x W^T + bias) + residual with
           8-bit rows and weights, a scale for each token and each channel
  loss     hsamp.cross_entropy: each row's loss (minus the log-probability of its
           token) over the whole vocabulary, without its logits
  grad     hsamp.cross_entropy_grad: its gradients of the rows and of the matrix
  embed    hsamp.embed: the tokens' rows of the matrix, scaled
  scatter  hsamp.embed_grad: the gradient of that, each token's rows added up

`run` computes the plain form of each with elementary torch operations, or,
where `own` is set, calls the library.
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

PKG_DIR = Path(__file__).resolve().parent.parent / "ultima.cpp_amd"
V_QWEN = 151936
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _hsamp():
    """ultima.cpp_amd's binding (the folder's name is no identifier)."""
    if "ultima_cpp_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "ultima_cpp_amd", PKG_DIR / "__init__.py", submodule_search_locations=[str(PKG_DIR)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ultima_cpp_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["ultima_cpp_amd"].hsamp


def listed():
    def i8(name, rows, inner, outer, act, dtype="bf16", out="same", groups=1, bias=True, residual=True, aligned=True):
        return dict(name=name, kind="i8", rows=rows, inner=inner, outer=outer, act=act, dtype=dtype, out=out,
                    groups=groups, bias=bias, residual=residual, aligned=aligned)

    def loss(name, kind, rows, inner, vocab, dtype="bf16", cap=0.0, ignored=0.0, aligned=True):
        return dict(name=name, kind=kind, rows=rows, inner=inner, vocab=vocab, dtype=dtype, cap=cap, ignored=ignored,
                    aligned=aligned)

    def embed(name, kind, tokens, width, vocab=V_QWEN, dtype="bf16", out="same", scale=1.0, ended=0.0, skew=0.0,
              aligned=True):
        return dict(name=name, kind=kind, tokens=tokens, width=width, vocab=vocab, dtype=dtype, out=out, scale=scale,
                    ended=ended, skew=skew, aligned=aligned)

    return [
        # a draft head's residual block on one token, its weight in 8 bits
        i8("i8_one", 1, 4096, 4096, "silu"),
        # four draft heads on a 64-slot step, one call
        i8("i8_heads", 64, 4096, 4096, "silu", groups=4),
        # the logits of 64 slots' blocks of five positions, capped
        i8("i8_logits", 320, 4096, V_QWEN, "softcap", out="f32", bias=False, residual=False),
        # a prompt's rows through a wide layer
        i8("i8_prompt", 4096, 4096, 16384, "gelu_tanh", dtype="f16"),
        # the log-probability of one session's token
        loss("loss_token", "loss", 1, 4096, V_QWEN),
        # the log-probabilities of a prompt's tokens
        loss("loss_prompt", "loss", 2048, 4096, V_QWEN),
        # a small head on a few ragged rows, some of them padding, logits capped; rows at odd addresses
        loss("grad_ragged", "grad", 301, 1002, 50257, dtype="f16", cap=30.0, ignored=0.2, aligned=False),
        # a training step's rows against the whole matrix
        loss("grad_train", "grad", 4096, 4096, V_QWEN),
        # the sampled tokens of a 64-slot step, some slots ended
        embed("embed_step", "embed", 64, 4096, ended=0.2),
        # a batch of prompts, scaled by the root of the width
        embed("embed_prompts", "embed", 16384, 4096, scale=64.0),
        # a short batch against a small odd vocabulary, float gradients
        embed("scatter_small", "scatter", 700, 1002, vocab=50257, dtype="f32", ended=0.1, aligned=False),
        # a training step's tokens, a few of them most of the text
        embed("scatter_train", "scatter", 32768, 4096, skew=1.1),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above."""
    kind = rng.choice(("i8", "i8", "loss", "grad", "embed", "scatter"))
    aligned = rng.random() < 0.75
    if kind == "i8":
        rows, groups = _log_int(rng, 1, 4096), rng.choice((1, 1, 1, 2, 5))
        inner = _log_int(rng, 64, 8192)
        outer = _log_int(rng, 64, max(65, min(V_QWEN, 4096 * 4096 * 16384 // (max(rows, 512) * inner * groups))))
        if aligned:
            inner, outer = max(64, inner // 64 * 64), max(16, outer // 16 * 16)
        return dict(kind=kind, rows=rows, inner=inner, outer=outer, groups=groups,
                    act=rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh", "softcap")),
                    dtype=rng.choice(("bf16", "f16")), out=rng.choice(("same", "f32")), bias=rng.random() < 0.6,
                    residual=rng.random() < 0.6, aligned=aligned)
    if kind in ("loss", "grad"):
        most = 2048 if kind == "loss" else 4096
        rows, inner = _log_int(rng, 1, most), _log_int(rng, 64, 8192)
        vocab = _log_int(rng, 1000, min(262144, max(1001, most * 4096 * V_QWEN // (2 * max(rows, 512) * inner))))
        if aligned:
            inner = max(64, inner // 64 * 64)
        return dict(kind=kind, rows=rows, inner=inner, vocab=vocab, dtype=rng.choice(("bf16", "f16")),
                    cap=rng.choice((0.0, 0.0, 30.0)), ignored=rng.choice((0.0, 0.3)), aligned=aligned)
    width = _log_int(rng, 64, 8192)
    if aligned:
        width = max(64, width // 64 * 64)
    vocab = _log_int(rng, 1000, min(262144, V_QWEN * 4096 // (2 * width)))
    tokens = _log_int(rng, 1, min(65536, (16384 if kind == "embed" else 32768) * 4096 // (2 * width)))
    return dict(kind=kind, tokens=tokens, width=width, vocab=vocab, dtype=rng.choice(("bf16", "f16", "f32")),
                out=rng.choice(("same", "f32")), scale=rng.choice((1.0, math.sqrt(width))),
                ended=rng.choice((0.0, 0.2)), skew=rng.choice((0.0, 1.1)), aligned=aligned)


# ---- inputs ------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & (2**62 - 1))
    i = {k: v for k, v in case.items() if k != "name"}
    dt = TYPES[case["dtype"]]
    pad = 0 if case["aligned"] else 3
    i["out_dtype"] = dt if case.get("out", "same") == "same" else TYPES[case["out"]]

    def normal(shape, scale, dtype=dt):
        buf = torch.empty((*shape[:-1], shape[-1] + pad), dtype=dtype, device="cuda")
        return buf.normal_(0.0, scale, generator=g)[..., :shape[-1]]

    def chosen(n, most):
        """Row numbers 0 .. most - 1, by Zipf's law where the case is skewed, -1 for ended ones."""
        if case.get("skew"):
            p = torch.arange(1, most + 1, device="cuda", dtype=torch.float64) ** -case["skew"]
            u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
            rank = torch.searchsorted(torch.cumsum(p, 0) / p.sum(), u).clamp(max=most - 1)
            ids = torch.randperm(most, generator=g, device="cuda")[rank]
        else:
            ids = torch.randint(0, most, (n,), generator=g, device="cuda")
        share = case.get("ended", case.get("ignored", 0.0))
        return torch.where(torch.rand(n, generator=g, device="cuda") < share, -1, ids).to(torch.int32)

    if case["kind"] == "i8":
        G, M, K, N = case["groups"], case["rows"], case["inner"], case["outer"]
        i["x"] = normal((M, K), 1.0)                      # the groups share their input
        # the weight as a program lays it out once: 8 bits and a scale per channel
        w = torch.empty((G, N, K + pad), dtype=torch.int8, device="cuda")
        i["ws"] = torch.empty((G, N), device="cuda")
        for k in range(G):
            f = torch.empty((N, K), device="cuda").normal_(0.0, K ** -0.5, generator=g)
            i["ws"][k] = f.abs().amax(1) / 127
            w[k, :, :K] = torch.round(f / i["ws"][k][:, None]).to(torch.int8)
        i["w"] = w[..., :K]
        i["b"] = normal((G, N), 0.5) if case["bias"] else None
        i["r"] = normal((G, M, N), 1.0) if case["residual"] else None
        return i
    if case["kind"] in ("loss", "grad"):
        M, K, V = case["rows"], case["inner"], case["vocab"]
        i["w"] = normal((V, K), 2.0 * K ** -0.5)
        i["t"] = chosen(M, V)
        # most rows point towards their token: its logit stands about ten above the rest
        x = torch.empty((M, K), device="cuda").normal_(0.0, 1.0, generator=g)
        sure = (torch.rand((M, 1), generator=g, device="cuda") < 0.7) * 2.5
        x += sure * i["w"][i["t"].clamp(min=0).long()].float()
        i["x"] = torch.empty((M, K + pad), dtype=dt, device="cuda")[:, :K].copy_(x)
        if case["kind"] == "grad":
            valid = i["t"] >= 0
            # the mean's gradient, rows weighted; half precision trains with a scaled loss
            up = (65536.0 if dt == torch.float16 else 1.0) / valid.sum().clamp(min=1)
            i["g"] = torch.where(valid, up * (0.5 + torch.rand(M, generator=g, device="cuda")), 0.0)
            i["lse"] = torch.empty(M, device="cuda")      # what the forward pass left
            for a in range(0, M, 512):
                i["lse"][a:a + 512] = torch.logsumexp(_logits(i, slice(a, a + 512)), 1)
        return i
    n, width, V = case["tokens"], case["width"], case["vocab"]
    i["t"] = chosen(n, V)
    if case["kind"] == "embed":
        i["w"] = normal((V, width), 1.0)
    else:
        i["d"] = normal((n, width), 1.0)
    return i


# ---- the calls and their plain forms --------------------------------------------------

def run(state):
    return {"i8": _i8, "loss": _loss, "grad": _grad, "embed": _embed, "scatter": _scatter}[state["kind"]](state)


def _i8(i):
    if own:
        hs = _hsamp()
        one = i["groups"] == 1
        take = lambda t: None if t is None else t[0] if one else t  # noqa: E731
        q, s = hs.quantize_rows(i["x"])
        if not one:
            q, s = q.expand(i["groups"], -1, -1), s.expand(i["groups"], -1)
        return {"y": hs.linear_i8(q, s, take(i["w"]), take(i["ws"]), bias=take(i["b"]), act=i["act"], act_param=30.0,
                                  residual=take(i["r"]), dtype=TYPES[i["dtype"]], out_dtype=i["out_dtype"])}
    x = i["x"].double()                                   # (half-way values are the exact quotient's)
    top = x.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(x * 127 / top), 0.0).float()
    y = torch.matmul(q, i["w"].float().transpose(-1, -2)) * (top / 127).float() * i["ws"][:, None, :]
    if i["b"] is not None:
        y = y + i["b"].float()[:, None, :]
    y = _act(y, i["act"])
    if i["r"] is not None:
        y = y + i["r"].float()
    y = y.to(i["out_dtype"])
    return {"y": y[0] if i["groups"] == 1 else y}


def _act(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "softcap":
        return 30.0 * torch.tanh(y / 30.0)
    return y


def _logits(i, rows=slice(None)):
    z = torch.matmul(i["x"][rows].float(), i["w"].float().t())
    return i["cap"] * torch.tanh(z / i["cap"]) if i["cap"] else z


def _loss(i):
    if own:
        out = _hsamp().cross_entropy(i["x"], i["w"], i["t"], softcap=i["cap"])
        return {"loss": out["loss"], "lse": out["lse"]}
    z = _logits(i)
    top = z.amax(1, keepdim=True)
    rest = torch.log(torch.exp(z - top).sum(1))
    at = z.gather(1, i["t"].clamp(min=0).long()[:, None])
    loss = torch.where(i["t"] >= 0, (top - at)[:, 0] + rest, 0.0)
    return {"loss": loss, "lse": top[:, 0] + rest}


def _grad(i):
    if own:
        out = _hsamp().cross_entropy_grad(i["x"], i["w"], i["t"], i["lse"], i["g"], softcap=i["cap"])
        return {"dx": out["d_x"], "dw": out["d_weight"]}
    z = _logits(i)
    d = torch.exp(z - i["lse"][:, None])
    row = torch.arange(i["rows"], device="cuda")
    d[row, i["t"].clamp(min=0).long()] -= (i["t"] >= 0).float()
    d *= torch.where(i["t"] >= 0, i["g"], 0.0)[:, None]
    if i["cap"]:
        d *= 1 - (z / i["cap"]) ** 2
    return {"dx": torch.matmul(d, i["w"].float()).to(i["x"].dtype),
            "dw": torch.matmul(d.t(), i["x"].float()).to(i["x"].dtype)}


def _embed(i):
    if own:
        return {"y": _hsamp().embed(i["w"], i["t"], scale=i["scale"], out_dtype=i["out_dtype"])}
    y = i["w"][i["t"].clamp(min=0).long()].float() * i["scale"]
    return {"y": torch.where((i["t"] >= 0)[:, None], y, 0.0).to(i["out_dtype"])}


def _scatter(i):
    if own:
        return {"dw": _hsamp().embed_grad(i["d"], i["t"], i["vocab"], scale=i["scale"], out_dtype=i["out_dtype"])}
    dw = torch.zeros((i["vocab"], i["width"]), device="cuda")
    d = torch.where((i["t"] >= 0)[:, None], i["d"].float() * i["scale"], 0.0)
    dw.index_add_(0, i["t"].clamp(min=0).long(), d)
    return {"dw": dw.to(i["out_dtype"])}


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    e = size[case["dtype"]]
    o = e if case.get("out", "same") == "same" else size[case["out"]]
    if case["kind"] == "i8":
        G, M, K, N = case["groups"], case["rows"], case["inner"], case["outer"]
        n = e * M * K + G * N * (K + 4) + G * M * N * (o + (e if case["residual"] else 0))
        return {"bytes": n + (e * G * N if case["bias"] else 0), "flops": 2.0 * G * M * N * K}
    if case["kind"] in ("loss", "grad"):
        M, K, V = case["rows"], case["inner"], case["vocab"]
        n, used = e * (M + V) * K + 12 * M, M * (1 - case["ignored"])
        if case["kind"] == "loss":
            return {"bytes": n, "flops": 2.0 * M * K * V}
        # the logits again, which nobody kept, and the two gradients; ignored rows need none of it
        return {"bytes": 2 * n, "flops": 6.0 * used * K * V}
    used = case["tokens"] * (1 - case["ended"])
    if case["kind"] == "embed":
        return {"bytes": case["width"] * (e * min(used, case["vocab"]) + o * case["tokens"]) + 4 * case["tokens"],
                "flops": case["width"] * used}
    return {"bytes": case["width"] * (e * used + o * case["vocab"]) + 4 * case["tokens"],
            "flops": case["width"] * used}


# ---- the same in 64 bits -------------------------------------------------------------

def exact(case, seed):
    i = prepare(case, seed)

    def i8():
        x = i["x"].double()
        top = x.abs().max(dim=1, keepdim=True).values.clamp(min=1e-300)
        x = (127 * x / top).round() * (top / 127)
        outs = []
        for g in range(i["groups"]):
            y = torch.empty((i["rows"], i["outer"]), dtype=torch.float64, device="cuda")
            for a in range(0, i["outer"], 8192):
                w = i["w"][g, a:a + 8192].double() * i["ws"][g, a:a + 8192, None].double()
                y[:, a:a + 8192] = x @ w.t().contiguous()
            if i["b"] is not None:
                y += i["b"][g].double()
            if i["act"] == "relu":
                y = y.relu()
            elif i["act"] == "silu":
                y = y * torch.sigmoid(y)
            elif i["act"] == "gelu":
                y = y * (1 - 0.5 * torch.erfc(y / 2 ** 0.5))
            elif i["act"] == "gelu_tanh":
                y = y * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3))
            elif i["act"] == "softcap":
                y = 30.0 * torch.tanh(y / 30.0)
            if i["r"] is not None:
                y += i["r"][g].double()
            outs.append(y)
        return {"y": outs[0] if i["groups"] == 1 else torch.stack(outs)}

    def loss():
        """A few rows at a time."""
        w = i["w"].double().t().contiguous()
        losses, sums = [], []
        for x, t in zip(i["x"].split(256), i["t"].split(256)):
            z = x.double() @ w
            if i["cap"]:
                z = i["cap"] * torch.tanh(z / i["cap"])
            lse = torch.logsumexp(z, 1)
            picked = torch.log_softmax(z, 1)[torch.arange(len(t), device="cuda"), t.long().clamp(min=0)]
            losses.append(torch.where(t < 0, torch.zeros_like(lse), -picked))
            sums.append(lse)
        return {"loss": torch.cat(losses), "lse": torch.cat(sums)}

    def grad():
        """A piece of the vocabulary at a time."""
        x, dx, dws = i["x"].double(), 0.0, []
        up = torch.where(i["t"] < 0, torch.zeros_like(i["g"]), i["g"]).double()
        for a in range(0, i["vocab"], 16384):
            w = i["w"][a:a + 16384].double()
            z = x @ w.t().contiguous()
            slope = torch.ones_like(z)
            if i["cap"]:
                z = i["cap"] * torch.tanh(z / i["cap"])
                slope = (1 + z / i["cap"]) * (1 - z / i["cap"])
            here = torch.arange(a, a + len(w), device="cuda")[None] == i["t"][:, None]
            dz = (torch.exp(z - i["lse"].double()[:, None]) - here.double()) * slope * up[:, None]
            dx = dx + dz @ w
            dws.append(dz.t().contiguous() @ x)
        return {"dx": dx, "dw": torch.cat(dws)}

    def embed():
        y = i["scale"] * torch.index_select(i["w"], 0, i["t"].clamp(min=0)).double()
        y[i["t"] < 0] = 0
        return {"y": y}

    def scatter():
        """Sorted tokens, differences of running sums at each token's ends."""
        t, order = torch.sort(i["t"], stable=True)
        total = torch.zeros((len(t) + 1, i["width"]), dtype=torch.float64, device="cuda")
        torch.cumsum(i["d"][order].double(), 0, out=total[1:])
        ids = torch.arange(i["vocab"], device="cuda", dtype=torch.int32)
        first, last = torch.searchsorted(t, ids), torch.searchsorted(t, ids, right=True)
        dw = total[last]
        dw -= total[first]
        return {"dw": dw * i["scale"]}

    return {"i8": i8, "loss": loss, "grad": grad, "embed": embed, "scatter": scatter}[i["kind"]]()
