"""ctypes binding of libultima_hsamp (include/ultima_hsamp.h).

PyTorch is used only to own device memory and streams; every sampling
decision is made by the library's HIP kernels. Loading fails loudly when the
library is not built.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

import numpy as np

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libultima_hsamp.so"
NOALLOC_LIB_PATH = PKG / "libultima_hsamp_noalloc.so"
HEADER = PKG.parent / "include" / "ultima_hsamp.h"
NOALLOC_HEADER = PKG.parent / "include" / "ultima_hsamp_noalloc.h"

OK, ERR_INVALID, ERR_HIP, ERR_UNSUPPORTED, ERR_NOMEM, ERR_CAPACITY, ERR_NO_DEVICE = 0, -1, -2, -3, -4, -5, -6
F32, BF16, F16 = 0, 1, 9
MAX_DRAFT = 1023
WRITEBACK, STREAM_ONLY = 1, 0x100
NOALLOC_SCRATCH_BYTES, NOALLOC_PLAN_BYTES = 96 << 20, 2 << 20
KERNELS_EXACT, KERNELS_GENERAL, KERNELS_FULL, KERNELS_WRITEBACK = 1, 2, 4, 8
ROW_GREEDY, ROW_U_USED, ROW_CDF_NEAR, ROW_NAN, ROW_UNIFORM, ROW_TOPP_NEAR, ROW_REREAD = 1, 2, 4, 8, 16, 32, 64

PARAM_KEYS = ("rep_penalty", "dry_multiplier", "dry_base", "frequency_penalty", "presence_penalty",
              "temperature", "top_p", "min_p", "repeat_last_n", "dry_allowed_len", "dry_last_n",
              "top_k")


class Params(ctypes.Structure):
    _fields_ = [
        ("rep_penalty", ctypes.c_float),
        ("dry_multiplier", ctypes.c_float),
        ("dry_base", ctypes.c_float),
        ("frequency_penalty", ctypes.c_float),
        ("presence_penalty", ctypes.c_float),
        ("temperature", ctypes.c_float),
        ("top_p", ctypes.c_float),
        ("min_p", ctypes.c_float),
        ("repeat_last_n", ctypes.c_uint64),
        ("dry_allowed_len", ctypes.c_uint64),
        ("dry_last_n", ctypes.c_uint64),
        ("top_k", ctypes.c_uint64),
        ("hist_len", ctypes.c_int64),
        ("bias_offset", ctypes.c_int64),
        ("bias_count", ctypes.c_int64),
    ]


class Batch(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("logits", ctypes.c_void_p),
        ("logits_stride", ctypes.c_int64),
        ("hist", ctypes.c_void_p),
        ("hist_stride", ctypes.c_int64),
        ("mask", ctypes.c_void_p),
        ("mask_stride", ctypes.c_int64),
        ("u", ctypes.c_void_p),
        ("params", ctypes.POINTER(Params)),
        ("bias_ids", ctypes.c_void_p),
        ("bias_vals", ctypes.c_void_p),
        ("token", ctypes.c_void_p),
        ("row_flags", ctypes.c_void_p),
        ("topk_idx", ctypes.c_void_p),
        ("topk_count", ctypes.c_void_p),
        ("kept_idx", ctypes.c_void_p),
        ("kept_prob", ctypes.c_void_p),
        ("kept_count", ctypes.c_void_p),
        ("set_cap", ctypes.c_int32),
        ("hist_len_dev", ctypes.c_void_p),
    ]


class Head(ctypes.Structure):
    """ultima_hsamp_head (include/ultima_hsamp.h)."""
    _fields_ = [
        ("hidden", ctypes.c_void_p),
        ("hidden_stride", ctypes.c_int64),
        ("rows", ctypes.c_int32),
        ("hidden_dim", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("weight_dtype", ctypes.c_int32),
        ("norm_scale", ctypes.c_void_p),
        ("eps", ctypes.c_float),
        ("logit_scale", ctypes.c_float),
        ("weight", ctypes.c_void_p),
        ("normed", ctypes.c_void_p),
        ("logits", ctypes.c_void_p),
        ("logits_stride", ctypes.c_int64),
        ("fold_block", ctypes.c_int32),
        ("fold_signs", ctypes.c_void_p),
    ]


class Commit(ctypes.Structure):
    """ultima_hsamp_commit (include/ultima_hsamp.h)."""
    _fields_ = [
        ("hist", ctypes.c_void_p),
        ("hist_stride", ctypes.c_int64),
        ("hist_len_dev", ctypes.c_void_p),
        ("active", ctypes.c_void_p),
        ("budget", ctypes.c_void_p),
        ("keep", ctypes.c_int32),
        ("n_stop", ctypes.c_int32),
        ("stop_ids", ctypes.c_void_p),
    ]


class Verify(ctypes.Structure):
    """ultima_hsamp_verify (include/ultima_hsamp.h)."""
    _fields_ = [
        ("n_pos", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("logits", ctypes.c_void_p),
        ("logits_stride", ctypes.c_int64),
        ("draft", ctypes.c_void_p),
        ("hist", ctypes.c_void_p),
        ("hist_len", ctypes.c_int32),
        ("mask", ctypes.c_void_p),
        ("mask_stride", ctypes.c_int64),
        ("u", ctypes.c_void_p),
        ("params", ctypes.POINTER(Params)),
        ("bias_ids", ctypes.c_void_p),
        ("bias_vals", ctypes.c_void_p),
        ("work", ctypes.c_void_p),
        ("out_tokens", ctypes.c_void_p),
        ("out_count", ctypes.c_void_p),
        ("row_flags", ctypes.c_void_p),
    ]


class Draft(ctypes.Structure):
    """ultima_hsamp_draft (include/ultima_hsamp.h)."""
    _fields_ = [
        ("seqs", ctypes.c_int32),
        ("max_draft", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("logits", ctypes.c_void_p),
        ("logits_stride", ctypes.c_int64),
        ("logits_rows", ctypes.c_int32),
        ("draft_rows", ctypes.c_int32),
        ("draft_logits", ctypes.c_void_p),
        ("draft_stride", ctypes.c_int64),
        ("draft", ctypes.c_void_p),
        ("n_draft", ctypes.c_void_p),
        ("target_start", ctypes.c_void_p),
        ("draft_start", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("draft_temperature", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("mask_stride", ctypes.c_int64),
        ("draft_mask", ctypes.c_void_p),
        ("draft_mask_stride", ctypes.c_int64),
        ("u_accept", ctypes.c_void_p),
        ("u_draw", ctypes.c_void_p),
        ("work", ctypes.c_void_p),
        ("out_tokens", ctypes.c_void_p),
        ("out_count", ctypes.c_void_p),
        ("accept_prob", ctypes.c_void_p),
    ]


class DraftSets(ctypes.Structure):
    """ultima_hsamp_draft_sets (include/ultima_hsamp.h)."""
    _fields_ = [
        ("seqs", ctypes.c_int32),
        ("max_draft", ctypes.c_int32),
        ("rows", ctypes.c_int32),
        ("draft_rows", ctypes.c_int32),
        ("kept_idx", ctypes.c_void_p),
        ("kept_prob", ctypes.c_void_p),
        ("kept_count", ctypes.c_void_p),
        ("set_cap", ctypes.c_int32),
        ("draft_cap", ctypes.c_int32),
        ("draft_idx", ctypes.c_void_p),
        ("draft_prob", ctypes.c_void_p),
        ("draft_count", ctypes.c_void_p),
        ("draft", ctypes.c_void_p),
        ("n_draft", ctypes.c_void_p),
        ("target_start", ctypes.c_void_p),
        ("draft_start", ctypes.c_void_p),
        ("u_accept", ctypes.c_void_p),
        ("u_draw", ctypes.c_void_p),
        ("work", ctypes.c_void_p),
        ("out_tokens", ctypes.c_void_p),
        ("out_count", ctypes.c_void_p),
        ("accept_prob", ctypes.c_void_p),
    ]


class LinearArgs(ctypes.Structure):
    """ultima_hsamp_linear_args (include/ultima_hsamp.h)."""
    _fields_ = [
        ("rows", ctypes.c_int32),
        ("in_dim", ctypes.c_int32),
        ("out_dim", ctypes.c_int32),
        ("groups", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("act", ctypes.c_int32),
        ("act_param", ctypes.c_float),
        ("x", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64),
        ("x_group", ctypes.c_int64),
        ("weight", ctypes.c_void_p),
        ("weight_stride", ctypes.c_int64),
        ("weight_group", ctypes.c_int64),
        ("bias", ctypes.c_void_p),
        ("bias_group", ctypes.c_int64),
        ("residual", ctypes.c_void_p),
        ("residual_stride", ctypes.c_int64),
        ("residual_group", ctypes.c_int64),
        ("out", ctypes.c_void_p),
        ("out_stride", ctypes.c_int64),
        ("out_group", ctypes.c_int64),
    ]


def declared_symbols(header: Path = HEADER) -> list[str]:
    """Function names declared in a header (default include/ultima_hsamp.h)."""
    import re
    text = header.read_text()
    return sorted(set(re.findall(r"\b(ultima_hsamp_[a-z_0-9]+)\s*\(", text)))


_lib = None


def lib() -> ctypes.CDLL:
    """Load libultima_hsamp.so. PyTorch-ROCm ships its own HIP runtime with the
    same SONAME as ROCm's; importing torch first makes the library bind to that
    one instance, since one process cannot hold two HSA runtimes."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is not built: run __graft_entry__.build()")
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(str(LIB_PATH))
        vp, i32, i64, f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_double
        L.ultima_hsamp_create.restype = ctypes.c_int
        L.ultima_hsamp_create.argtypes = [ctypes.c_int, i32, i32, ctypes.POINTER(vp)]
        L.ultima_hsamp_destroy.restype = ctypes.c_int
        L.ultima_hsamp_destroy.argtypes = [vp]
        L.ultima_hsamp_run.restype = ctypes.c_int
        L.ultima_hsamp_run.argtypes = [vp, ctypes.POINTER(Batch), vp]
        L.ultima_hsamp_sample_host.restype = ctypes.c_int
        L.ultima_hsamp_sample_host.argtypes = [vp, vp, i32, ctypes.POINTER(Params), vp, vp, vp, f64,
                                               ctypes.c_int, ctypes.POINTER(i32)]
        L.ultima_hsamp_params_default.restype = None
        L.ultima_hsamp_params_default.argtypes = [ctypes.POINTER(Params)]
        L.ultima_hsamp_params_identity.restype = None
        L.ultima_hsamp_params_identity.argtypes = [ctypes.POINTER(Params)]
        L.ultima_hsamp_uniform_from_u64.restype = f64
        L.ultima_hsamp_uniform_from_u64.argtypes = [ctypes.c_uint64]
        L.ultima_hsamp_status_str.restype = ctypes.c_char_p
        L.ultima_hsamp_status_str.argtypes = [ctypes.c_int]
        L.ultima_hsamp_version.restype = ctypes.c_int
        L.ultima_hsamp_version.argtypes = []
        L.ultima_hsamp_query_kernels.restype = ctypes.c_int
        L.ultima_hsamp_query_kernels.argtypes = [vp, ctypes.POINTER(Batch), ctypes.POINTER(ctypes.c_uint32)]
        L.ultima_hsamp_read_probe.restype = ctypes.c_int
        L.ultima_hsamp_read_probe.argtypes = [vp, ctypes.POINTER(Batch), vp, vp]
        L.ultima_hsamp_set_phase_event.restype = ctypes.c_int
        L.ultima_hsamp_set_phase_event.argtypes = [vp, vp]
        L.ultima_hsamp_history_push.restype = ctypes.c_int
        L.ultima_hsamp_history_push.argtypes = [vp, ctypes.c_int64, vp, vp, i32, i32, vp]
        L.ultima_hsamp_lm_head.restype = ctypes.c_int
        L.ultima_hsamp_lm_head.argtypes = [ctypes.POINTER(Head), vp]
        L.ultima_hsamp_decode_commit.restype = ctypes.c_int
        L.ultima_hsamp_decode_commit.argtypes = [vp, i64, vp, vp, vp, vp, i32, i32, vp, i32, vp]
        L.ultima_hsamp_run_commit.restype = ctypes.c_int
        L.ultima_hsamp_run_commit.argtypes = [vp, ctypes.POINTER(Batch), ctypes.POINTER(Commit), vp]
        L.ultima_hsamp_verify_work_ints.restype = i64
        L.ultima_hsamp_verify_work_ints.argtypes = [i32, i32]
        L.ultima_hsamp_verify_block.restype = ctypes.c_int
        L.ultima_hsamp_verify_block.argtypes = [vp, ctypes.POINTER(Verify), vp]
        L.ultima_hsamp_verify_draft_work_bytes.restype = i64
        L.ultima_hsamp_verify_draft_work_bytes.argtypes = [i32, i32, i32]
        L.ultima_hsamp_verify_draft.restype = ctypes.c_int
        L.ultima_hsamp_verify_draft.argtypes = [ctypes.POINTER(Draft), vp]
        L.ultima_hsamp_verify_sets_work_bytes.restype = i64
        L.ultima_hsamp_verify_sets_work_bytes.argtypes = [i32, i32]
        L.ultima_hsamp_verify_sets.restype = ctypes.c_int
        L.ultima_hsamp_verify_sets.argtypes = [ctypes.POINTER(DraftSets), vp]
        L.ultima_hsamp_linear.restype = ctypes.c_int
        L.ultima_hsamp_linear.argtypes = [ctypes.POINTER(LinearArgs), vp]
        _lib = L
    return _lib


class HsampError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {status} ({lib().ultima_hsamp_status_str(status).decode()})")


def check(status: int, what: str) -> None:
    if status != OK:
        raise HsampError(status, what)


def make_params(plist, hist_len=None, bias=None):
    """(ctypes array of Params, bias ids array, bias values array) for a list of
    knob dicts. bias: list (per row) of {id: value} or None."""
    B = len(plist)
    arr = (Params * B)()
    ids, vals = [], []
    for r, p in enumerate(plist):
        q = arr[r]
        for k in PARAM_KEYS:
            setattr(q, k, p[k])
        q.hist_len = 0 if hist_len is None else int(hist_len[r])
        q.bias_offset = len(ids)
        b = bias[r] if bias is not None else None
        q.bias_count = 0 if not b else len(b)
        if b:
            for t, v in b.items():
                ids.append(int(t))
                vals.append(float(v))
    bids = np.array(ids, np.int32) if ids else None
    bvals = np.array(vals, np.float32) if vals else None
    return arr, bids, bvals


def _batch(logits, params, u, hist, hist_len, mask, bias, writeback, want_sets, set_cap, stream, outputs,
           stream_only, hist_len_dev=None):
    """An ultima_hsamp_batch over torch tensors: (batch, outputs, host arrays
    the call reads, stream)."""
    import torch
    B, V = logits.shape[0], logits.shape[1]
    dev = logits.device
    out = outputs if outputs is not None else {}
    if "token" not in out:
        out["token"] = torch.empty(B, dtype=torch.int32, device=dev)
    if "row_flags" not in out:
        out["row_flags"] = torch.empty(B, dtype=torch.int32, device=dev)
    cap = 0
    if want_sets:
        cap = set_cap or V
        for k, dt in (("topk_idx", torch.int32), ("kept_idx", torch.int32),
                      ("kept_prob", torch.float32)):
            if k not in out:
                out[k] = torch.empty((B, cap), dtype=dt, device=dev)
        for k in ("topk_count", "kept_count"):
            if k not in out:
                out[k] = torch.empty(B, dtype=torch.int32, device=dev)
    parr, bids, bvals = make_params(params, hist_len, bias)
    b = Batch()
    b.rows, b.vocab = B, V
    b.dtype = F32 if logits.dtype == torch.float32 else BF16
    b.flags = (WRITEBACK if writeback else 0) | (STREAM_ONLY if stream_only else 0)
    b.logits = logits.data_ptr()
    b.logits_stride = logits.stride(0)
    if hist is not None:
        b.hist = hist.data_ptr()
        b.hist_stride = hist.stride(0)
    if hist_len_dev is not None:
        b.hist_len_dev = hist_len_dev.data_ptr()
    if mask is not None:
        b.mask = mask.data_ptr()
        b.mask_stride = mask.stride(0)
    b.u = u.data_ptr()
    b.params = ctypes.cast(parr, ctypes.POINTER(Params))
    if bids is not None:
        b.bias_ids = bids.ctypes.data
        b.bias_vals = bvals.ctypes.data
    b.token = out["token"].data_ptr()
    b.row_flags = out["row_flags"].data_ptr()
    if want_sets:
        b.topk_idx = out["topk_idx"].data_ptr()
        b.topk_count = out["topk_count"].data_ptr()
        b.kept_idx = out["kept_idx"].data_ptr()
        b.kept_prob = out["kept_prob"].data_ptr()
        b.kept_count = out["kept_count"].data_ptr()
        b.set_cap = cap
    elif "kept_count" in out:
        b.kept_count = out["kept_count"].data_ptr()   # the count alone
    s = torch.cuda.current_stream(dev) if stream is None else stream
    return b, out, (parr, bids, bvals), s


_noalloc_lib = None


def noalloc_lib() -> ctypes.CDLL:
    """Load libultima_hsamp_noalloc.so (include/ultima_hsamp_noalloc.h); it
    links libultima_hsamp.so, loaded first."""
    global _noalloc_lib
    if _noalloc_lib is None:
        lib()
        if not NOALLOC_LIB_PATH.exists():
            raise RuntimeError(f"{NOALLOC_LIB_PATH} is not built: run __graft_entry__.build()")
        L = ctypes.CDLL(str(NOALLOC_LIB_PATH))
        L.ultima_hsamp_run_noalloc.restype = ctypes.c_int
        L.ultima_hsamp_run_noalloc.argtypes = [ctypes.POINTER(Batch), ctypes.c_void_p]
        _noalloc_lib = L
    return _noalloc_lib


def run_noalloc(logits, params, u, hist=None, hist_len=None, mask=None, bias=None, writeback=False,
                want_sets=False, set_cap=None, stream=None, outputs=None):
    """ultima_hsamp_run_noalloc on the current device: Sampler.run without a
    handle, scratch from the library's fixed device array."""
    b, out, keep, s = _batch(logits, params, u, hist, hist_len, mask, bias, writeback, want_sets, set_cap,
                             stream, outputs, False)
    check(noalloc_lib().ultima_hsamp_run_noalloc(ctypes.byref(b), ctypes.c_void_p(s.cuda_stream)), "run_noalloc")
    del keep
    return out


def history_push(hist, hist_len_dev, tokens, keep: int, stream=None) -> None:
    """ultima_hsamp_history_push on torch tensors of one device: hist int32
    [rows, stride] (the rows' histories), hist_len_dev int32 [rows] (their
    lengths, advanced here), tokens int32 [rows] (appended; e.g. the token
    output of run()). A full row first keeps its last `keep` ids."""
    import torch
    rows = hist.shape[0]
    assert hist.dtype == torch.int32 and hist_len_dev.dtype == torch.int32 and tokens.dtype == torch.int32
    assert hist_len_dev.shape[0] >= rows and tokens.shape[0] >= rows and hist.stride(1) == 1
    s = torch.cuda.current_stream(hist.device) if stream is None else stream
    check(lib().ultima_hsamp_history_push(ctypes.c_void_p(hist.data_ptr()), hist.stride(0),
                                          ctypes.c_void_p(hist_len_dev.data_ptr()),
                                          ctypes.c_void_p(tokens.data_ptr()), rows, int(keep),
                                          ctypes.c_void_p(s.cuda_stream)), "history_push")


def decode_commit(hist, hist_len_dev, tokens, active, keep: int, stop_ids=(), budget=None, stream=None) -> None:
    """ultima_hsamp_decode_commit on torch tensors of one device (int32): after
    a run() over the slots' rows, ends the rows whose token is a stop id (or
    -1), marks the tokens of ended rows -1, appends the rest to the histories
    and counts them against budget (the server loop's max_tokens)."""
    import torch
    rows = hist.shape[0]
    for t in (hist, hist_len_dev, tokens, active) + ((budget,) if budget is not None else ()):
        assert t.dtype == torch.int32 and t.device == hist.device
    assert hist_len_dev.shape[0] >= rows and tokens.shape[0] >= rows and active.shape[0] >= rows
    assert hist.stride(1) == 1 and (budget is None or budget.shape[0] >= rows)
    stop = np.asarray(list(stop_ids), np.int32)
    s = torch.cuda.current_stream(hist.device) if stream is None else stream
    check(lib().ultima_hsamp_decode_commit(
        ctypes.c_void_p(hist.data_ptr()), hist.stride(0), ctypes.c_void_p(hist_len_dev.data_ptr()),
        ctypes.c_void_p(tokens.data_ptr()), ctypes.c_void_p(active.data_ptr()),
        ctypes.c_void_p(budget.data_ptr() if budget is not None else 0), rows, int(keep),
        stop.ctypes.data_as(ctypes.c_void_p) if stop.size else None, int(stop.size),
        ctypes.c_void_p(s.cuda_stream)), "decode_commit")


# head weight types (ULTIMA_HSAMP_F32 / _BF16 / _HEAD_*)
HEAD_Q4_K, HEAD_Q5_K, HEAD_Q6_K, HEAD_Q8_0, HEAD_Q4_1, HEAD_Q5_0, HEAD_PQ2_0 = range(2, 9)


def lm_head(hidden, norm_scale, eps: float, weight, logit_scale: float = 1.0, logits=None, normed=None,
            stream=None, weight_dtype=None, fold_block: int = 0, fold_signs=None):
    """ultima_hsamp_lm_head on torch tensors of one device: hidden [rows, H] f32,
    norm_scale [H] f32, weight [V, H] f32 or bf16, or a quantised head [V, row
    bytes] uint8 with weight_dtype one of HEAD_Q*; fold_block / fold_signs [H]
    f32 the Hadamard fold. Returns (logits [rows, V], normed [rows, H]); the
    outputs may be passed in (allocated otherwise)."""
    import torch
    if hidden.dim() == 1:
        hidden = hidden.unsqueeze(0)
    rows, H = hidden.shape
    V = weight.shape[0]
    dev = hidden.device
    if weight_dtype is None:
        if weight.dtype not in (torch.float32, torch.bfloat16):
            raise HsampError(ERR_INVALID, "lm_head: weight must be float32 or bfloat16 (or give weight_dtype)")
        weight_dtype = BF16 if weight.dtype == torch.bfloat16 else F32
    if logits is None:
        logits = torch.empty((rows, V), dtype=torch.float32, device=dev)
    if normed is None:
        normed = torch.empty((rows, H), dtype=torch.float32, device=dev)
    h = Head()
    h.hidden = hidden.data_ptr()
    h.hidden_stride = hidden.stride(0)
    h.rows, h.hidden_dim, h.vocab = rows, H, V
    h.weight_dtype = weight_dtype
    h.norm_scale = norm_scale.data_ptr()
    h.eps = eps
    h.logit_scale = logit_scale
    h.weight = weight.data_ptr()
    h.normed = normed.data_ptr()
    h.logits = logits.data_ptr()
    h.logits_stride = logits.stride(0)
    h.fold_block = fold_block
    h.fold_signs = None if fold_signs is None else fold_signs.data_ptr()
    s = torch.cuda.current_stream(dev) if stream is None else stream
    check(lib().ultima_hsamp_lm_head(ctypes.byref(h), ctypes.c_void_p(s.cuda_stream)), "lm_head")
    return logits, normed


def _refuse(what: str):
    raise HsampError(ERR_INVALID, what)


def _elsewhere(dev, stream, what):
    """The context that makes `stream` (None: the device's current one) and its device
    current, or None where they are: the call, and what it allocates, then go there."""
    import torch
    if stream is not None:
        if stream.device != dev:
            _refuse(f"{what}: the stream must be one of {dev}")
        return torch.cuda.stream(stream)
    return None if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _used_on(stream, *tensors):
    """Their memory is not handed out again before `stream` is done with what it has."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _launch(fn, a, dev, what):
    import torch
    status = fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(dev.index))
    if status != OK:
        raise HsampError(status, what)


def _vector(t, n, dtype, dev, what, name):
    """The address of a contiguous vector of n (None: any number) elements, or None."""
    if t is None:
        return None
    if t.dtype != dtype or t.device != dev or t.dim() != 1 or (n is not None and t.shape[0] != n) or not t.is_contiguous():
        _refuse(f"{what}: {name} must be a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {dev}")
    return t.data_ptr()


def _rows(t, n, width, dtypes, dev, what, name):
    """The address and row stride of n rows of at least `width` elements."""
    if t.dtype not in dtypes or t.device != dev or t.dim() != 2 or t.shape[0] != n or t.shape[1] < width or \
            (t.shape[1] > 1 and t.stride(1) != 1):
        _refuse(f"{what}: {name} must be {n} rows of {width} {dtypes[0]} on {dev}")
    return t.data_ptr(), t.stride(0) if n > 1 else max(width, t.stride(0))


def _seq_args(a, what, dev, draft, u_accept, u_draw, max_draft, n_draft, target_start, draft_start, accept, outputs):
    """The fields of Draft and DraftSets that say which rows are whose."""
    import torch
    i32, f64 = torch.int32, torch.float64
    if u_draw is None:
        _refuse(f"{what}: u_draw is missing")
    a.u_draw, at = _vector(u_draw, None, f64, dev, what, "u_draw"), _vector(draft, None, i32, dev, what, "draft")
    B, K, D = u_draw.shape[0], int(max_draft), 0 if draft is None else draft.shape[0]
    if B < 1 or not 0 <= K <= MAX_DRAFT or (u_accept is None) != (draft is None):
        _refuse(f"{what}: at least one sequence, max_draft 0 .. {MAX_DRAFT}, draft and u_accept together")
    u = _vector(u_accept, D, f64, dev, what, "u_accept")
    a.seqs, a.max_draft, a.draft_rows = B, K, D
    if D:
        a.draft, a.u_accept = at, u
    a.n_draft = _vector(n_draft, B, i32, dev, what, "n_draft")
    a.target_start = _vector(target_start, B, i32, dev, what, "target_start")
    a.draft_start = _vector(draft_start, B, i32, dev, what, "draft_start")
    out = {} if outputs is None else outputs
    for name, shape, dt in (("tokens", (B, K + 1), i32), ("count", (B,), i32), ("accept", (D,), torch.float32)):
        t = out.get(name)
        if t is None:
            if name != "accept" or accept:
                out[name] = torch.empty(shape, dtype=dt, device=dev)
        elif t.shape != shape or t.dtype != dt or t.device != dev or not t.is_contiguous():
            _refuse(f"{what}: output {name} must be contiguous {dt} {shape} on {dev}")
    a.out_tokens, a.out_count = out["tokens"].data_ptr(), out["count"].data_ptr()
    if D and "accept" in out:
        a.accept_prob = out["accept"].data_ptr()
    return out


def _work(work, need, dev, what):
    """The caller's scratch, looked over, or scratch of the current stream."""
    import torch
    if work is None:
        return torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    if work.device != dev or not work.is_contiguous() or work.numel() * work.element_size() < need:
        _refuse(f"{what}: work must be {need} contiguous bytes on {dev}")
    return work


def verify_draft(logits, draft, u_accept, u_draw, max_draft: int, draft_logits=None, temperature=None,
                 draft_temperature=None, mask=None, draft_mask=None, n_draft=None, target_start=None,
                 draft_start=None, accept: bool = True, work=None, outputs=None, stream=None):
    """ultima_hsamp_verify_draft on torch tensors of one device: drafted tokens
    (int32 [D]) against the target's logits [R, V] and the drafter's [D, V] (None:
    certain drafts), float32 or bfloat16, by the rejection rule. u_accept f64 [D],
    u_draw f64 [B]; temperature, draft_temperature f32 [B] (None: 1; <= 0:
    greedy); mask, draft_mask int32 words per row; n_draft, target_start,
    draft_start int32 [B] for sequences of different lengths. Returns a dict:
    tokens int32 [B, max_draft + 1], count int32 [B] and, unless accept is False,
    accept f32 [D] (their acceptance probabilities; drafted rows of no sequence, and
    of sequences whose n_draft or rows are out of range, are not written: what they
    hold is then no probability). work: a uint8 tensor of
    ultima_hsamp_verify_draft_work_bytes() bytes of this call alone (allocated
    otherwise); outputs: a dict of tensors to write to; stream: a stream of their
    device to run on instead of the current one (it has to wait for what makes the
    tensors; their memory is kept until it is done with this call)."""
    import torch
    what, f32 = "verify_draft", torch.float32
    dev = logits.device
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in (f32, torch.bfloat16):
        _refuse("verify_draft: logits must be a float32 or bfloat16 matrix on the GPU")
    there = _elsewhere(dev, stream, what)
    if there is not None:
        with there:
            out = verify_draft(logits, draft, u_accept, u_draw, max_draft, draft_logits, temperature, draft_temperature,
                               mask, draft_mask, n_draft, target_start, draft_start, accept, work, outputs)
        _used_on(stream, logits, draft, u_accept, u_draw, draft_logits, temperature, draft_temperature, mask, draft_mask,
                 n_draft, target_start, draft_start, work, *out.values())
        return out
    rows, V = logits.shape
    a = Draft()
    out = _seq_args(a, what, dev, draft, u_accept, u_draw, max_draft, n_draft, target_start, draft_start, accept,
                    outputs)
    D, B = a.draft_rows, a.seqs
    a.vocab, a.dtype, a.logits_rows = V, F32 if logits.dtype == f32 else BF16, rows
    a.logits, a.logits_stride = _rows(logits, rows, V, (logits.dtype,), dev, what, "logits")
    if draft_logits is not None:
        at, stride = _rows(draft_logits, D, V, (logits.dtype,), dev, what, "draft_logits")
        if draft_logits.shape[1] != V:
            _refuse("verify_draft: draft_logits must have the target's vocabulary")
        if D:
            a.draft_logits, a.draft_stride = at, stride
    words, kinds = -(-V // 32), (torch.int32, torch.uint32)
    if mask is not None:
        a.mask, a.mask_stride = _rows(mask, rows, words, kinds, dev, what, "mask")
    if draft_mask is not None:
        at, stride = _rows(draft_mask, D, words, kinds, dev, what, "draft_mask")
        if draft_logits is None:
            _refuse("verify_draft: draft_mask goes with draft_logits")
        if D:
            a.draft_mask, a.draft_mask_stride = at, stride
    a.temperature = _vector(temperature, B, f32, dev, what, "temperature")
    a.draft_temperature = _vector(draft_temperature, B, f32, dev, what, "draft_temperature")
    work = _work(work, lib().ultima_hsamp_verify_draft_work_bytes(B, a.max_draft, V), dev, what)
    a.work = work.data_ptr()
    _launch(lib().ultima_hsamp_verify_draft, a, dev, what)
    return out


def verify_sets(kept_idx, kept_prob, kept_count, draft, u_accept, u_draw, max_draft: int, draft_idx=None,
                draft_prob=None, draft_count=None, n_draft=None, target_start=None, draft_start=None,
                accept: bool = True, work=None, outputs=None, stream=None):
    """ultima_hsamp_verify_sets on torch tensors of one device: drafted tokens
    against the kept sets that run() leaves for the target's rows (kept_idx int32
    [R, cap], kept_prob f32 [R, cap], kept_count int32 [R]) and, unless the drafts
    are certain, for the drafter's. The other arguments and the result as in
    verify_draft; work: ultima_hsamp_verify_sets_work_bytes() bytes."""
    import torch
    what = "verify_sets"
    dev = kept_idx.device
    if not kept_idx.is_cuda or kept_idx.dim() != 2:
        _refuse("verify_sets: kept_idx must be a matrix on the GPU")
    there = _elsewhere(dev, stream, what)
    if there is not None:
        with there:
            out = verify_sets(kept_idx, kept_prob, kept_count, draft, u_accept, u_draw, max_draft, draft_idx, draft_prob,
                              draft_count, n_draft, target_start, draft_start, accept, work, outputs)
        _used_on(stream, kept_idx, kept_prob, kept_count, draft, u_accept, u_draw, draft_idx, draft_prob, draft_count,
                 n_draft, target_start, draft_start, work, *out.values())
        return out

    def sets(idx, prob, count, rows, names):
        if prob is None or count is None or idx.dtype != torch.int32 or prob.dtype != torch.float32 or \
                count.dtype != torch.int32 or idx.dim() != 2 or idx.shape[0] != rows or prob.shape != idx.shape or \
                count.shape != (rows,) or not (idx.device == prob.device == count.device == dev) or \
                not (idx.is_contiguous() and prob.is_contiguous() and count.is_contiguous()):
            _refuse(f"{what}: {names} must be contiguous int32 [{rows}, cap], float32 [{rows}, cap], int32 [{rows}] on {dev}")
        return idx.data_ptr(), prob.data_ptr(), count.data_ptr()

    a = DraftSets()
    out = _seq_args(a, what, dev, draft, u_accept, u_draw, max_draft, n_draft, target_start, draft_start, accept,
                    outputs)
    a.rows, a.set_cap = kept_idx.shape
    a.kept_idx, a.kept_prob, a.kept_count = sets(kept_idx, kept_prob, kept_count, a.rows,
                                                 "kept_idx, kept_prob, kept_count")
    if draft_idx is not None:
        at = sets(draft_idx, draft_prob, draft_count, a.draft_rows, "draft_idx, draft_prob, draft_count")
        if a.draft_rows:
            a.draft_cap = draft_idx.shape[1]
            a.draft_idx, a.draft_prob, a.draft_count = at
    elif draft_prob is not None or draft_count is not None:
        _refuse("verify_sets: draft_prob and draft_count go with draft_idx")
    need = lib().ultima_hsamp_verify_sets_work_bytes(a.seqs, a.set_cap)
    if need > 0 or work is not None:
        work = _work(work, need, dev, what)
        a.work = work.data_ptr()
    _launch(lib().ultima_hsamp_verify_sets, a, dev, what)
    return out


ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "softcap": 5}


def _matrix(t, lead, rows, columns, dtype, dev, name):
    """The address, row stride and group stride of a [*lead, rows, columns] operand."""
    shape, stride = t.shape, t.stride()
    if shape[:-2] != lead or len(shape) < 2 or shape[-2] != rows or shape[-1] != columns or t.dtype != dtype or \
            t.device != dev or (columns > 1 and stride[-1] != 1):
        _refuse(f"linear: {name} must be {dtype} {(*lead, rows, columns)} on {dev}, contiguous in its last dimension")
    return t.data_ptr(), stride[-2] if rows > 1 else max(columns, stride[-2]), stride[0] if lead else 0


def linear(x, weight, bias=None, act: str = "none", act_param: float = 0.0, residual=None, out=None, out_dtype=None,
           stream=None):
    """ultima_hsamp_linear on torch tensors of one device: act(x weight^T + bias)
    + residual, x [M, K] and weight [N, K], or with a leading dimension of groups
    on all of them (expanded dimensions are fine); bfloat16 or float16, the output
    in that type or in float32 (out_dtype; out: the tensor to write, which may be
    the residual). act: one of ACTS; act_param: the cap of "softcap"; stream: as in
    verify_draft."""
    import torch
    dev, dt = x.device, x.dtype
    if not x.is_cuda or dt not in (torch.bfloat16, torch.float16) or x.dim() not in (2, 3) or weight.dim() != x.dim():
        _refuse("linear: x and weight must be bfloat16 or float16 matrices (or batches of them) on the GPU")
    if act not in ACTS:
        _refuse(f"linear: act must be one of {', '.join(ACTS)}")
    there = _elsewhere(dev, stream, "linear")
    if there is not None:
        with there:
            out = linear(x, weight, bias, act, act_param, residual, out, out_dtype)
        _used_on(stream, x, weight, bias, residual, out)
        return out
    lead = x.shape[:-2]
    M, K = x.shape[-2:]
    N = weight.shape[-2]
    if out is None:
        out = torch.empty((*lead, M, N), dtype=out_dtype or dt, device=dev)
    odt = out.dtype
    if odt not in (dt, torch.float32) or out_dtype not in (None, odt):
        _refuse(f"linear: the output must be {dt} or torch.float32")
    kind = BF16 if dt == torch.bfloat16 else F16
    a = LinearArgs(M, K, N, lead[0] if lead else 1, kind, F32 if odt == torch.float32 else kind, ACTS[act], act_param)
    a.x, a.x_stride, a.x_group = _matrix(x, lead, M, K, dt, dev, "x")
    a.weight, a.weight_stride, a.weight_group = _matrix(weight, lead, N, K, dt, dev, "weight")
    if bias is not None:
        if bias.shape != (*lead, N) or bias.dtype != dt or bias.device != dev or (N > 1 and bias.stride(-1) != 1):
            _refuse(f"linear: bias must be {dt} {(*lead, N)} on {dev}, contiguous in its last dimension")
        a.bias, a.bias_group = bias.data_ptr(), bias.stride(0) if lead else 0
    if residual is not None:
        a.residual, a.residual_stride, a.residual_group = _matrix(residual, lead, M, N, dt, dev, "residual")
    a.out, a.out_stride, a.out_group = _matrix(out, lead, M, N, odt, dev, "out")
    _launch(lib().ultima_hsamp_linear, a, dev, "linear")
    return out


class Sampler:
    """A handle on one device (create/destroy of the C ABI)."""

    def __init__(self, device: int = 0, max_rows: int = 1024, max_vocab: int = 1 << 18):
        self.device = device
        h = ctypes.c_void_p()
        check(lib().ultima_hsamp_create(device, max_rows, max_vocab, ctypes.byref(h)), "create")
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            lib().ultima_hsamp_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def run(self, logits, params, u, hist=None, hist_len=None, mask=None, bias=None,
            writeback=False, want_sets=False, set_cap=None, stream=None, outputs=None, stream_only=False,
            hist_len_dev=None):
        """Sample every row. logits: cuda tensor [B, >=V] float32 or bfloat16
        (row stride = logits.stride(0)); u: cuda float64 [B]; hist: cuda int32
        [B, H]; mask: cuda int32/uint32 [B, W]. Returns a dict of cuda tensors.
        `outputs` may carry preallocated tensors (token, row_flags, ...).
        stream_only (diagnostics): run only the pass over the logits.
        hist_len_dev: cuda int32 [B], the rows' history lengths read on the
        device (a history kept by history_push)."""
        b, out, keep, s = _batch(logits, params, u, hist, hist_len, mask, bias, writeback, want_sets, set_cap,
                                 stream, outputs, stream_only, hist_len_dev)
        check(lib().ultima_hsamp_run(self.h, ctypes.byref(b), ctypes.c_void_p(s.cuda_stream)), "run")
        del keep
        return out

    def batch(self, logits, params, u, hist=None, hist_len=None, mask=None, bias=None, outputs=None):
        """The ultima_hsamp_batch run() would pass for these tensors: (batch,
        host arrays it points into, which the caller keeps alive). For callers
        that time the C ABI itself (bench.py's uncaptured figure)."""
        b, out, keep, s = _batch(logits, params, u, hist, hist_len, mask, bias, False, False, None, None,
                                 outputs, False)
        return b, (out, keep)

    def read_probe(self, logits, params, u, out, hist=None, hist_len=None, mask=None, stream=None):
        """Diagnostics: a plain read of `logits` with the launch shape run()
        would use (ultima_hsamp_read_probe); out: cuda float32, rows * 256."""
        import torch
        b, _, keep, s = _batch(logits, params, u, hist, hist_len, mask, None, False, False, None, stream,
                               {"token": out, "row_flags": out}, False)
        check(lib().ultima_hsamp_read_probe(self.h, ctypes.byref(b), ctypes.c_void_p(out.data_ptr()),
                                            ctypes.c_void_p(s.cuda_stream)), "read_probe")
        del keep, torch

    def query_kernels(self, logits, params, u, hist=None, hist_len=None, mask=None, bias=None,
                      writeback=False) -> int:
        """ultima_hsamp_query_kernels: the KERNELS_* bits of the kernels run()
        would launch for this batch (nothing is launched)."""
        b, _, keep, _s = _batch(logits, params, u, hist, hist_len, mask, bias, writeback, False, None, None,
                                None, False)
        k = ctypes.c_uint32(0)
        check(lib().ultima_hsamp_query_kernels(self.h, ctypes.byref(b), ctypes.byref(k)), "query_kernels")
        del keep
        return int(k.value)

    def set_phase_event(self, event):
        """Record `event` (a torch.cuda.Event already recorded once, or None)
        between the stream and merge kernels of every later run()."""
        ptr = None if event is None else ctypes.c_void_p(event.cuda_event)
        check(lib().ultima_hsamp_set_phase_event(self.h, ptr), "set_phase_event")

    def run_commit(self, logits, params, u, hist, hist_len, hist_len_dev, active, keep: int, stop_ids=(),
                   budget=None, mask=None, bias=None, outputs=None, stream=None):
        """ultima_hsamp_run_commit: run() over the rows' device histories
        (hist int32 [rows, stride], hist_len_dev int32 [rows]) with
        decode_commit's rules applied where each token is decided."""
        import torch
        b, out, keep_alive, s = _batch(logits, params, u, hist, hist_len, mask, bias, False, False, None, stream,
                                       outputs, False, hist_len_dev=hist_len_dev)
        stop = np.asarray(list(stop_ids), np.int32)
        c = Commit()
        c.hist, c.hist_stride, c.hist_len_dev = hist.data_ptr(), hist.stride(0), hist_len_dev.data_ptr()
        c.active = active.data_ptr()
        c.budget = budget.data_ptr() if budget is not None else None
        c.keep, c.n_stop = int(keep), int(stop.size)
        c.stop_ids = stop.ctypes.data if stop.size else None
        check(lib().ultima_hsamp_run_commit(self.h, ctypes.byref(b), ctypes.byref(c), ctypes.c_void_p(s.cuda_stream)),
              "run_commit")
        self._keep = (keep_alive, stop)
        return out

    def verify_block(self, logits, params: dict, u, draft=None, hist=None, mask=None, bias=None, stream=None):
        """ultima_hsamp_verify_block on torch tensors of one device: logits
        [n_pos, V] (each position's target logits), u f64 [n_pos], draft int32
        [n_pos - 1], hist int32 [hist_len] (the sequence's ids before the
        block), one knob dict. Returns (tokens int32 [n_pos], count int32 [1],
        row_flags int32 [n_pos]): the loop's emitted tokens are tokens[:count]."""
        import torch
        n, V = logits.shape[0], logits.shape[1]
        dev = logits.device
        dt = {torch.float32: F32, torch.bfloat16: BF16}[logits.dtype]
        assert logits.stride(1) == 1 and u.dtype == torch.float64 and u.shape[0] >= n
        assert draft is None or (draft.dtype == torch.int32 and draft.shape[0] >= n - 1)
        assert hist is None or hist.dtype == torch.int32
        L = 0 if hist is None else int(hist.shape[0])
        arr, bids, bvals = make_params([params], None, None if bias is None else [bias])
        work = torch.empty(int(lib().ultima_hsamp_verify_work_ints(n, L)), dtype=torch.int32, device=dev)
        toks = torch.empty(n, dtype=torch.int32, device=dev)
        count = torch.empty(1, dtype=torch.int32, device=dev)
        flags = torch.empty(n, dtype=torch.int32, device=dev)
        v = Verify()
        v.n_pos, v.vocab, v.dtype = n, V, dt
        v.logits, v.logits_stride = logits.data_ptr(), logits.stride(0)
        v.draft = draft.data_ptr() if draft is not None and n > 1 else None
        v.hist = hist.data_ptr() if L > 0 else None
        v.hist_len = L
        if mask is not None:
            v.mask, v.mask_stride = mask.data_ptr(), mask.stride(0)
        v.u = u.data_ptr()
        v.params = arr
        v.bias_ids = bids.ctypes.data if bids is not None else None
        v.bias_vals = bvals.ctypes.data if bvals is not None else None
        v.work, v.out_tokens, v.out_count, v.row_flags = work.data_ptr(), toks.data_ptr(), count.data_ptr(), flags.data_ptr()
        s = torch.cuda.current_stream(dev) if stream is None else stream
        check(lib().ultima_hsamp_verify_block(self.h, ctypes.byref(v), ctypes.c_void_p(s.cuda_stream)), "verify_block")
        self._keep = (arr, bids, bvals, work)   # read on the host during the call only; work until it completes
        return toks, count, flags

    def sample_host(self, logits: np.ndarray, params: dict, hist=None, bias=None, u: float = 0.5,
                    writeback: bool = False):
        """One host row (sample() with an explicit uniform). Returns (token, logits)."""
        x = np.array(logits, dtype=np.float32, copy=True)
        h = None if hist is None else np.ascontiguousarray(hist, dtype=np.int32)
        parr, bids, bvals = make_params([params], [0 if h is None else h.size], [bias] if bias else None)
        tok = ctypes.c_int32(-1)
        check(lib().ultima_hsamp_sample_host(
            self.h, x.ctypes.data, x.size, parr, None if h is None else h.ctypes.data,
            None if bids is None else bids.ctypes.data, None if bvals is None else bvals.ctypes.data,
            float(u), 1 if writeback else 0, ctypes.byref(tok)), "sample_host")
        return int(tok.value), x
