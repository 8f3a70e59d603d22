"""The operators of speculative decoding, as timed cases.

Three operators, each through the call a serving program makes of it:

  draft   hsamp.verify_draft: drafted tokens against the target's and the
          drafter's logits by the rejection rule
  sets    hsamp.verify_sets: the same on the kept sets (ids and probabilities
          after top-k, top-p, min-p) that the sampler writes
  linear  hsamp.linear: act(x W^T + bias) + residual

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
    def draft(name, seqs, drafts, vocab, dtype, drafter=True, ragged=False, mask=False, greedy=False):
        return dict(name=name, kind="draft", seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype, drafter=drafter,
                    ragged=ragged, mask=mask, greedy=greedy)

    def sets(name, seqs, drafts, cap, vocab=V_QWEN, drafter=True, ragged=False):
        return dict(name=name, kind="sets", seqs=seqs, drafts=drafts, cap=cap, vocab=vocab, drafter=drafter,
                    ragged=ragged)

    def linear(name, rows, inner, outer, act, dtype="bf16", out="bf16", groups=1, bias=True, residual=True,
               aligned=True):
        return dict(name=name, kind="linear", rows=rows, inner=inner, outer=outer, act=act, dtype=dtype, out=out,
                    groups=groups, bias=bias, residual=residual, aligned=aligned)

    return [
        # one interactive session, four tokens drafted: latency
        draft("draft_one", 1, 4, V_QWEN, "f32"),
        # a 64-slot server's step, four tokens drafted per slot
        draft("draft_slots", 64, 4, V_QWEN, "f32"),
        # slots that drafted different numbers of tokens, a small odd vocabulary in bf16 (rows at odd addresses)
        draft("draft_ragged", 37, 7, 50257, "bf16", ragged=True),
        # tokens copied from the prompt (no drafter), a grammar's mask, some slots greedy
        draft("draft_lookup", 16, 15, V_QWEN, "f32", drafter=False, mask=True, greedy=True),
        # a large batch of long drafts
        draft("draft_batch", 256, 8, V_QWEN, "bf16"),
        # one session whose sampler keeps at most 64 ids
        sets("sets_one", 1, 4, 64),
        # a 64-slot step, top-k up to 1000
        sets("sets_slots", 64, 8, 1024, ragged=True),
        # nucleus sets over the whole vocabulary, tens of thousands of ids
        sets("sets_nucleus", 32, 4, 32768),
        # a draft head's residual block on one token
        linear("linear_one", 1, 4096, 4096, "silu"),
        # four draft heads on a 64-slot step, one call
        linear("linear_heads", 64, 4096, 4096, "silu", groups=4),
        # the logits of 64 slots' blocks of five positions, capped
        linear("linear_logits", 320, 4096, V_QWEN, "softcap", out="f32", bias=False, residual=False),
        # a prompt's rows through a wide layer
        linear("linear_prompt", 4096, 4096, 16384, "gelu_tanh", dtype="f16", out="f16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above."""
    kind = rng.choice(("draft", "sets", "linear", "linear"))
    if kind == "draft":
        vocab = _log_int(rng, 2000, 262144)
        drafts = rng.randint(1, 16)
        most = max(1, 256 * 17 * V_QWEN // (2 * vocab * (2 * drafts + 1)))
        return dict(kind="draft", seqs=_log_int(rng, 1, min(256, most)), drafts=drafts, vocab=vocab,
                    dtype=rng.choice(("f32", "bf16")), drafter=rng.random() < 0.7, ragged=rng.random() < 0.5,
                    mask=rng.random() < 0.3, greedy=rng.random() < 0.4)
    if kind == "sets":
        vocab = _log_int(rng, 2000, 262144)
        cap = min(vocab, _log_int(rng, 8, 32768))
        return dict(kind="sets", seqs=_log_int(rng, 1, max(1, min(256, 32 * 32768 // cap))), drafts=rng.randint(1, 8),
                    cap=cap, vocab=vocab, drafter=rng.random() < 0.7, ragged=rng.random() < 0.5)
    rows, groups = _log_int(rng, 1, 4096), rng.choice((1, 1, 1, 2, 5))
    inner = _log_int(rng, 64, 8192)
    outer = _log_int(rng, 64, max(65, min(V_QWEN, 4096 * 4096 * 16384 // (max(rows, 512) * inner * groups))))
    if rng.random() < 0.75:
        inner = max(64, inner // 64 * 64)
        outer = max(16, outer // 16 * 16)
    return dict(kind="linear", rows=rows, inner=inner, outer=outer, groups=groups,
                act=rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh", "softcap")),
                dtype=rng.choice(("bf16", "f16")), out=rng.choice(("same", "f32")), bias=rng.random() < 0.6,
                residual=rng.random() < 0.6, aligned=rng.random() < 0.8)


# ---- inputs ------------------------------------------------------------------------

def _lengths(case, g):
    """Drafted tokens per sequence, and where each sequence's rows begin."""
    B, K = case["seqs"], case["drafts"]
    if not case["ragged"]:
        return None, None, None, B * (K + 1), B * K
    # 0 .. K tokens, as often as each other, in any order (the total is the same for every seed)
    n = (torch.randperm(B, generator=g, device="cuda") % (K + 1)).to(torch.int32)
    ts = (torch.cumsum(n + 1, 0) - n - 1).to(torch.int32)
    ds = (torch.cumsum(n, 0) - n).to(torch.int32)
    total = int(n.sum())
    return n, ts, ds, total + B, max(1, total)


def _mask(rows, vocab, g):
    """Allowed-token words (about a tenth of the ids) and the same as booleans."""
    words = -(-vocab // 32)
    ok = torch.rand((rows, words * 32), generator=g, device="cuda") < 0.1
    ok[:, vocab:] = False
    ok.scatter_(1, torch.randint(0, vocab, (rows, 1), generator=g, device="cuda"), True)
    bit = torch.ones((), dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    w = (ok.view(rows, words, 32) * bit).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32), ok[:, :vocab]


def _rows_of(i):
    """Per sequence: its drafted tokens, its first target row, its first drafted row."""
    B, K, dev = i["seqs"], i["drafts"], "cuda"
    n = torch.full((B,), K, dtype=torch.int32, device=dev) if i["n"] is None else i["n"]
    ts = torch.arange(B, device=dev) * (K + 1) if i["ts"] is None else i["ts"].long()
    ds = torch.arange(B, device=dev) * K if i["ds"] is None else i["ds"].long()
    return n.long(), ts, ds


def _target_rows_of_drafts(i):
    """The target row of every drafted row."""
    n, ts, ds = _rows_of(i)
    at = torch.zeros(i["draft_rows"], dtype=torch.int64, device="cuda")
    k = torch.arange(i["drafts"], device="cuda")
    real = k[None, :] < n[:, None]
    at[(ds[:, None] + k)[real]] = (ts[:, None] + k)[real]
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & (2**62 - 1))
    i = {k: v for k, v in case.items() if k != "name"}
    if case["kind"] == "linear":
        dt = {"bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]]
        G, M, K, N = case["groups"], case["rows"], case["inner"], case["outer"]
        pad = 0 if case["aligned"] else 3

        def normal(shape, scale):
            buf = torch.empty((*shape[:-1], shape[-1] + pad), dtype=dt, device="cuda")
            return buf.normal_(0.0, scale, generator=g)[..., :shape[-1]]

        i["x"] = normal((M, K), 1.0)                      # the groups share their input
        i["w"] = normal((G, N, K), K ** -0.5)
        i["b"] = normal((G, N), 0.5) if case["bias"] else None
        i["r"] = normal((G, M, N), 1.0) if case["residual"] else None
        i["out_dtype"] = {"f32": torch.float32, "same": dt, "bf16": torch.bfloat16, "f16": torch.float16}[case["out"]]
        return i
    B, K, V = case["seqs"], case["drafts"], case["vocab"]
    i["n"], i["ts"], i["ds"], rows, drows = _lengths(case, g)
    i["rows"], i["draft_rows"] = rows, drows
    i["u"] = torch.rand(drows, generator=g, device="cuda", dtype=torch.float64)
    i["v"] = torch.rand(B, generator=g, device="cuda", dtype=torch.float64)
    at = _target_rows_of_drafts(i)
    dt = torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32
    # a long tail, and a few likely tokens a row
    x = torch.empty((rows, V), device="cuda").normal_(0.0, 2.5, generator=g)
    x.scatter_(1, torch.randint(0, V, (rows, 6), generator=g, device="cuda"),
               torch.empty((rows, 6), device="cuda").normal_(13.0, 2.0, generator=g))
    y = x[at] + torch.empty((drows, V), device="cuda").normal_(0.0, 0.5, generator=g)
    if case["kind"] == "draft":
        i["ok"] = i["mask"] = None
        if case["mask"]:
            i["mask"], i["ok"] = _mask(rows, V, g)
        i["t"] = torch.rand(B, generator=g, device="cuda") * 0.6 + 0.4
        if case["greedy"]:
            i["t"][::3] = 0.0
        i["td"] = torch.rand(B, generator=g, device="cuda") * 0.6 + 0.4
        i["x"], i["y"] = x.to(dt), y.to(dt)
        # the drafts are the drafter's samples; without a drafter, often the target's likeliest token
        z = i["y"].float() / 0.7
        if i["ok"] is not None:
            z.masked_fill_(~i["ok"][at], -math.inf)
        noise = torch.empty_like(z).exponential_(generator=g).log_()
        if not case["drafter"]:
            noise *= torch.rand((drows, 1), generator=g, device="cuda") > 0.7
        z -= noise
        i["d"] = z.argmax(1).to(torch.int32)
        if not case["drafter"]:
            i["y"] = None
        return i
    # sets: the most likely ids of each row, between one and cap of them, by id
    cap = case["cap"]

    def kept(z):
        count = torch.randint(1, cap + 1, (z.shape[0],), generator=g, device="cuda", dtype=torch.int32)
        count[::2] = torch.clamp(count[::2], min=cap // 2 + 1)
        val, idx = torch.topk(z, cap, dim=1)
        val = val.masked_fill(torch.arange(cap, device="cuda")[None] >= count[:, None], -math.inf)
        p = torch.softmax(val / 0.8, 1)
        idx, order = torch.sort(torch.where(val > -math.inf, idx, V), dim=1)
        return idx.to(torch.int32), p.gather(1, order).contiguous(), count

    i["pi"], i["pp"], i["pc"] = kept(x)
    i["qi"], i["qp"], i["qc"] = kept(y)
    pick = torch.multinomial(i["qp"], 1, generator=g)
    i["d"] = i["qi"].gather(1, pick)[:, 0].contiguous()
    if not case["drafter"]:
        i["qi"] = i["qp"] = i["qc"] = None
    return i


# ---- the calls and their plain forms --------------------------------------------------

def run(state):
    return {"draft": _draft, "sets": _sets, "linear": _linear}[state["kind"]](state)


def _linear(i):
    if own:
        hs = _hsamp()
        x = i["x"] if i["groups"] == 1 else i["x"].expand(i["groups"], -1, -1)
        one = i["groups"] == 1
        take = lambda t: None if t is None else t[0] if one else t  # noqa: E731
        return {"y": hs.linear(x, take(i["w"]), bias=take(i["b"]), act=i["act"], act_param=30.0,
                               residual=take(i["r"]), out_dtype=i["out_dtype"])}
    y = torch.matmul(i["x"].float(), i["w"].float().transpose(-1, -2))
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


def _accept(i, p_d, q_d):
    """From the drafted rows' p(d) and q(d): the accepted counts and the
    acceptance probabilities (-1 after a sequence's first rejection)."""
    n, _, ds = _rows_of(i)
    k = torch.arange(i["drafts"], device="cuda")
    real = k[None, :] < n[:, None]
    row = torch.where(real, ds[:, None] + k, 0)
    ok = (i["u"] * q_d < p_d)[row] & real
    m = torch.cumprod(ok.long(), 1).sum(1)
    a = torch.full((i["draft_rows"],), -1.0, dtype=torch.float32, device="cuda")
    seen = real & (k[None, :] <= m[:, None])
    share = torch.where(p_d < q_d, p_d / q_d, torch.where(p_d > 0, 1.0, 0.0)).float()
    a[row[seen]] = share[row[seen]]
    d = i["d"][row]
    head = torch.where(k[None, :] < m[:, None], d, -1)
    return n, m, a, torch.cat([head, torch.full_like(head[:, :1], -1)], 1)


def _pick(r, p, v):
    """The lowest place whose running sum reaches v times the whole, of r (of p where r is empty)."""
    r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
    c = torch.cumsum(r, 1)
    good = (r > 0) & (c >= v[:, None] * c[:, -1:])
    place = torch.arange(r.shape[1], device="cuda")
    last = torch.where(r > 0, place, -1).amax(1)
    return torch.minimum(torch.where(good, place, r.shape[1]).amin(1), last)


def _chances(x, t, ok):
    """softmax(x / t) in 64 bits, t <= 0: all on the lowest of the largest."""
    z = x.double()
    if ok is not None:
        z = z.masked_fill(~ok, -math.inf)
    top = z.amax(1, keepdim=True)
    t = t.double()[:, None]
    e = torch.exp((z - top) / torch.where(t > 0, t, 1.0))
    place = torch.arange(z.shape[1], device="cuda")
    first = torch.where(z == top, place, z.shape[1]).amin(1, keepdim=True)
    e = torch.where(t > 0, e, (place[None] == first).double())
    return e / e.sum(1, keepdim=True)


def _draft(i):
    if own:
        out = _hsamp().verify_draft(i["x"], i["d"], i["u"], i["v"], i["drafts"], draft_logits=i["y"],
                                    temperature=i["t"], draft_temperature=i["td"] if i["y"] is not None else None,
                                    mask=i["mask"], n_draft=i["n"], target_start=i["ts"], draft_start=i["ds"])
        return {"tokens": out["tokens"], "count": out["count"], "accept": out["accept"]}
    n, ts, ds = _rows_of(i)
    at = _target_rows_of_drafts(i)
    seq = torch.zeros(i["rows"], dtype=torch.int64, device="cuda")
    k = torch.arange(i["drafts"] + 1, device="cuda")
    real = k[None, :] <= n[:, None]
    seq[(ts[:, None] + k)[real]] = torch.arange(i["seqs"], device="cuda")[:, None].expand_as(real)[real]
    p = _chances(i["x"], i["t"][seq], i["ok"])
    d = i["d"].long()[:, None]
    p_d = p[at].gather(1, d)[:, 0]
    q = None if i["y"] is None else _chances(i["y"], i["td"][seq[at]], None)
    q_d = torch.ones_like(p_d) if q is None else q.gather(1, d)[:, 0]
    n, m, accept, tokens = _accept(i, p_d, q_d)
    p_m = p[ts + m]
    row = torch.where(m < n, ds + m, 0)
    q_m = torch.zeros_like(p_m).scatter_(1, d[row], 1.0) if q is None else q[row]
    r = torch.where((m < n)[:, None], torch.clamp(p_m - q_m, min=0), p_m)
    tokens.scatter_(1, m[:, None], _pick(r, p_m, i["v"]).to(torch.int32)[:, None])
    return {"tokens": tokens, "count": (m + 1).to(torch.int32), "accept": accept}


def _sets(i):
    if own:
        out = _hsamp().verify_sets(i["pi"], i["pp"], i["pc"], i["d"], i["u"], i["v"], i["drafts"], draft_idx=i["qi"],
                                   draft_prob=i["qp"], draft_count=i["qc"], n_draft=i["n"], target_start=i["ts"],
                                   draft_start=i["ds"])
        return {"tokens": out["tokens"], "count": out["count"], "accept": out["accept"]}
    n, ts, ds = _rows_of(i)
    at = _target_rows_of_drafts(i)
    place = torch.arange(i["cap"], device="cuda")[None]
    d = i["d"][:, None]
    p_d = torch.where((i["pi"][at] == d) & (place < i["pc"][at][:, None]), i["pp"][at].double(), 0.0).sum(1)
    q_d = torch.ones_like(p_d)
    if i["qi"] is not None:
        q_d = torch.where((i["qi"] == d) & (place < i["qc"][:, None]), i["qp"].double(), 0.0).sum(1)
    n, m, accept, tokens = _accept(i, p_d, q_d)
    here = ts + m
    p = torch.where(place < i["pc"][here][:, None], i["pp"][here].double(), 0.0)
    row = torch.where(m < n, ds + m, 0)
    dense = torch.zeros((i["seqs"], i["vocab"] + 1), dtype=torch.float64, device="cuda")
    if i["qi"] is None:
        dense.scatter_(1, d[row].long(), 1.0)
    else:
        inside = place < i["qc"][row][:, None]
        dense.scatter_(1, torch.where(inside, i["qi"][row].long(), i["vocab"]), i["qp"][row].double())
    q = dense.gather(1, i["pi"][here].long())
    r = torch.where((m < n)[:, None], torch.clamp(p - q, min=0), p)
    r = torch.where(place < i["pc"][here][:, None], r, 0.0)
    token = i["pi"][here].gather(1, _pick(r, p, i["v"])[:, None])
    tokens.scatter_(1, m[:, None], token)
    return {"tokens": tokens, "count": (m + 1).to(torch.int32), "accept": accept}


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    if case["kind"] == "linear":
        G, M, K, N = case["groups"], case["rows"], case["inner"], case["outer"]
        out = 4 if case["out"] == "f32" else 2
        n = 2 * (M * K + G * N * K) + G * M * N * (out + (2 if case["residual"] else 0)) + (2 * G * N if case["bias"] else 0)
        return {"bytes": n, "flops": 2.0 * G * M * N * K}
    B = case["seqs"]
    drafted = B * case["drafts"] // (2 if case["ragged"] else 1)   # ragged: half of them, on average
    small = B * (case["drafts"] + 4) * 4 + drafted * 16
    if case["kind"] == "draft":
        rows = drafted + B + (drafted if case["drafter"] else 0)
        n = rows * case["vocab"] * (4 if case["dtype"] == "f32" else 2)
        n += (drafted + B) * (-(-case["vocab"] // 32)) * 4 if case["mask"] else 0
        return {"bytes": n + small, "flops": 4.0 * rows * case["vocab"]}
    # a search in each set, and one position's two sets whole (about five eighths of the capacity filled)
    sides = 2 if case["drafter"] else 1
    each = case["cap"] * 5 // 8
    return {"bytes": sides * (B * each * 8 + drafted * 4 * math.ceil(math.log2(case["cap"] + 1))) + small,
            "flops": 4.0 * B * each}


# ---- the same in 64 bits -------------------------------------------------------------

def exact(case, seed):
    i = prepare(case, seed)

    def linear():
        outs = []
        for g in range(i["groups"]):
            y = torch.empty((i["rows"], i["outer"]), dtype=torch.float64, device="cuda")
            for a in range(0, i["outer"], 8192):
                y[:, a:a + 8192] = i["x"].double() @ i["w"][g, a:a + 8192].double().t().contiguous()
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

    def chances(side, row, seq):
        """The distribution of one row as a dense 64-bit vector."""
        p = torch.zeros(i["vocab"], dtype=torch.float64, device="cuda")
        if i["kind"] == "sets":
            idx, prob, count = (i[side + k] for k in ("i", "p", "c"))
            c = int(count[row])
            p[idx[row, :c].long()] = prob[row, :c].double()
            return p
        z = (i["x"] if side == "p" else i["y"])[row].double()
        t = float((i["t"] if side == "p" else i["td"])[seq])
        if side == "p" and i["ok"] is not None:
            z = torch.where(i["ok"][row], z, torch.full_like(z, -math.inf))
        if t <= 0:
            p[int((z == z.max()).nonzero()[0, 0])] = 1.0
            return p
        return torch.softmax(z / t, 0)

    def verify():
        """One sequence after the other, one position after the other."""
        B, K = i["seqs"], i["drafts"]
        n, ts, ds = (t.tolist() for t in _rows_of(i))
        d, u, v = i["d"].tolist(), i["u"].tolist(), i["v"].tolist()
        drafter = (i["y"] if i["kind"] == "draft" else i["qi"]) is not None
        tokens = torch.full((B, K + 1), -1, dtype=torch.int32)
        count = torch.zeros(B, dtype=torch.int32)
        accept = torch.full((i["draft_rows"],), -1.0, dtype=torch.float64)
        for b in range(B):
            for k in range(n[b] + 1):
                r = p = chances("p", ts[b] + k, b)
                if k < n[b]:
                    at, token = ds[b] + k, d[ds[b] + k]
                    if drafter:
                        q = chances("q", at, b)
                    else:
                        q = torch.zeros_like(p)
                        q[token] = 1.0
                    p_d, q_d = p[token].item(), q[token].item()
                    accept[at] = min(1.0, p_d / q_d) if q_d > 0 else float(p_d > 0)
                    if u[at] * q_d < p_d:
                        tokens[b, k] = token
                        continue
                    r = torch.relu(p - q)
                    r = r if r.sum() > 0 else p
                at = r.nonzero()[:, 0]
                c = torch.cumsum(r[at], 0)
                first = min(int((c < v[b] * c[-1]).sum()), at.numel() - 1)
                tokens[b, k] = int(at[first])
                count[b] = k + 1
                break
        return {"tokens": tokens, "count": count, "accept": accept}

    return linear() if case["kind"] == "linear" else verify()
