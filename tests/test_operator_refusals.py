"""What verify_draft, verify_sets and linear refuse, through the C ABI and without
a GPU: every call here returns before anything is launched."""
import ctypes

import pytest

OK_PTR = 1 << 20      # never looked at: the call is refused first


@pytest.fixture(scope="module")
def hsamp(pkg):
    return pkg.hsamp


def draft(hsamp, **kw):
    a = hsamp.Draft()
    a.seqs, a.max_draft, a.vocab, a.dtype = 2, 3, 100, hsamp.F32
    a.logits, a.logits_stride, a.logits_rows, a.draft_rows = OK_PTR, 100, 8, 6
    a.draft_logits, a.draft_stride = OK_PTR, 100
    for k in ("draft", "u_accept", "u_draw", "work", "out_tokens", "out_count"):
        setattr(a, k, OK_PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return hsamp.lib().ultima_hsamp_verify_draft(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(seqs=0), dict(seqs=-1), dict(max_draft=-1), dict(max_draft=1024), dict(vocab=0), dict(vocab=(1 << 24) + 1),
    dict(dtype=2), dict(dtype=9), dict(dtype=-1), dict(logits=None), dict(logits_stride=99), dict(logits_rows=7),
    dict(logits_rows=0), dict(draft_rows=5), dict(draft_rows=-1), dict(draft_stride=99), dict(draft=None),
    dict(u_accept=None), dict(u_draw=None), dict(work=None), dict(work=OK_PTR + 8), dict(out_tokens=None),
    dict(out_count=None), dict(mask=OK_PTR, mask_stride=3), dict(draft_mask=OK_PTR, draft_mask_stride=3),
    dict(draft_logits=None, draft_mask=OK_PTR, draft_mask_stride=4), dict(seqs=3), dict(logits=OK_PTR + 2),
    dict(draft_logits=OK_PTR + 1), dict(draft_start=OK_PTR, logits_rows=7),
])
def test_draft_refuses(hsamp, kw):
    assert draft(hsamp, **kw) == hsamp.ERR_INVALID


def test_draft_refuses_null_and_too_much(hsamp):
    assert hsamp.lib().ultima_hsamp_verify_draft(None, None) == hsamp.ERR_INVALID
    # more blocks than a launch counts
    assert draft(hsamp, seqs=1 << 20, max_draft=100, target_start=OK_PTR, draft_start=OK_PTR) == hsamp.ERR_UNSUPPORTED
    assert draft(hsamp, seqs=2**31 - 1, max_draft=1023, vocab=1 << 24, logits_stride=1 << 24, draft_stride=1 << 24,
                 target_start=OK_PTR, draft_start=OK_PTR) == hsamp.ERR_UNSUPPORTED


def test_draft_work_bytes(hsamp):
    f = hsamp.lib().ultima_hsamp_verify_draft_work_bytes
    assert f(0, 1, 10) == -1 and f(1, -1, 10) == -1 and f(1, 1024, 10) == -1 and f(1, 1, 0) == -1
    assert f(1, 1, (1 << 24) + 1) == -1
    assert 0 < f(1, 0, 1) <= f(1, 1, 1) <= f(2, 1, 1) <= f(2, 1, 151936)
    assert f(2**31 - 1, 1023, 1 << 24) > 2**40      # no 32-bit overflow


def sets(hsamp, **kw):
    a = hsamp.DraftSets()
    a.seqs, a.max_draft, a.rows, a.draft_rows, a.set_cap, a.draft_cap = 2, 3, 8, 6, 64, 32
    for k in ("kept_idx", "kept_prob", "kept_count", "draft_idx", "draft_prob", "draft_count", "draft", "u_accept",
              "u_draw", "out_tokens", "out_count"):
        setattr(a, k, OK_PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return hsamp.lib().ultima_hsamp_verify_sets(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(seqs=0), dict(max_draft=-1), dict(max_draft=1024), dict(rows=0), dict(rows=7), dict(draft_rows=5),
    dict(draft_rows=-1), dict(set_cap=0), dict(set_cap=(1 << 24) + 1), dict(draft_cap=0), dict(draft_cap=(1 << 24) + 1),
    dict(kept_idx=None), dict(kept_prob=None), dict(kept_count=None), dict(draft_idx=None), dict(draft_prob=None),
    dict(draft_count=None), dict(draft=None), dict(u_accept=None), dict(u_draw=None), dict(out_tokens=None),
    dict(out_count=None), dict(set_cap=4097), dict(set_cap=4097, work=OK_PTR + 8),
])
def test_sets_refuse(hsamp, kw):
    assert sets(hsamp, **kw) == hsamp.ERR_INVALID


def test_sets_work_bytes(hsamp):
    f = hsamp.lib().ultima_hsamp_verify_sets_work_bytes
    assert f(0, 1) == -1 and f(1, 0) == -1 and f(1, (1 << 24) + 1) == -1
    assert f(1, 1) == f(5, 4096) == 0 < f(1, 4097) < f(2, 4097) < f(2, 151936)
    assert f(2**31 - 1, 1 << 24) > 2**40      # no 32-bit overflow


def test_sets_refuse_too_many(hsamp):
    assert sets(hsamp, seqs=(1 << 21) + 1, target_start=OK_PTR, draft_start=OK_PTR) == hsamp.ERR_UNSUPPORTED


def test_sets_refuse_null(hsamp):
    assert hsamp.lib().ultima_hsamp_verify_sets(None, None) == hsamp.ERR_INVALID


def linear(hsamp, **kw):
    a = hsamp.LinearArgs()
    a.rows, a.in_dim, a.out_dim, a.groups, a.dtype, a.out_dtype = 4, 64, 32, 2, hsamp.BF16, hsamp.BF16
    a.x, a.weight, a.bias, a.residual, a.out = (OK_PTR * k for k in (1, 2, 3, 4, 5))
    a.x_stride = a.weight_stride = 64
    a.residual_stride = a.out_stride = 32
    a.weight_group, a.residual_group, a.out_group = 64 * 32, 128, 128
    for k, v in kw.items():
        setattr(a, k, v)
    return hsamp.lib().ultima_hsamp_linear(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(rows=-1), dict(in_dim=0), dict(out_dim=0), dict(groups=0), dict(dtype=0), dict(dtype=2),
    dict(out_dtype=9), dict(out_dtype=2), dict(act=-1), dict(act=6), dict(act=5), dict(act=5, act_param=-1.0),
    dict(act=5, act_param=float("nan")), dict(act=5, act_param=float("inf")), dict(x=None), dict(weight=None),
    dict(out=None), dict(x_stride=63), dict(weight_stride=63), dict(out_stride=31), dict(residual_stride=31),
    dict(x=OK_PTR + 1), dict(weight=OK_PTR + 1), dict(bias=OK_PTR + 1), dict(residual=OK_PTR + 1), dict(out=OK_PTR + 1),
    dict(out_dtype=0, out=OK_PTR + 2), dict(out=OK_PTR), dict(out=2 * OK_PTR), dict(out=3 * OK_PTR),
    dict(residual=OK_PTR * 5, out_stride=33), dict(residual=OK_PTR * 5, out_dtype=0), dict(residual=OK_PTR * 5, out_group=256),
    dict(out_group=0), dict(out_group=64), dict(out_group=-1), dict(out_group=-64), dict(out_group=31, out_stride=64),
    dict(out_group=40, out_stride=64), dict(out_group=1 << 62, groups=0),
])
def test_linear_refuses(hsamp, kw):
    assert linear(hsamp, **kw) == hsamp.ERR_INVALID


def test_linear_refuses_null_and_too_much(hsamp):
    assert hsamp.lib().ultima_hsamp_linear(None, None) == hsamp.ERR_INVALID
    big = 1 << 31
    assert linear(hsamp, groups=65536) == hsamp.ERR_UNSUPPORTED
    assert linear(hsamp, groups=1, in_dim=(1 << 30) + 1, x_stride=big, weight_stride=big) == hsamp.ERR_UNSUPPORTED
    assert linear(hsamp, groups=1, out_dim=(1 << 30) + 1, residual_stride=big, out_stride=big) == hsamp.ERR_UNSUPPORTED
    assert linear(hsamp, groups=1, rows=(1 << 30) + 1) == hsamp.ERR_UNSUPPORTED
    assert linear(hsamp, groups=1, rows=1 << 30, out_dim=4096, residual_stride=4096, out_stride=4096) == hsamp.ERR_UNSUPPORTED
    assert linear(hsamp, groups=1, rows=1, out_dim=1 << 27, residual_stride=big, out_stride=big) == hsamp.ERR_UNSUPPORTED


def test_bindings_match_the_header(hsamp):
    """The ctypes structures have the C ones' sizes (a compiled sizeof)."""
    import subprocess
    import tempfile
    from pathlib import Path
    src = '#include <stdio.h>\n#include "ultima_hsamp.h"\nint main(void) { printf("%zu %zu %zu\\n", ' \
          'sizeof(ultima_hsamp_draft), sizeof(ultima_hsamp_draft_sets), sizeof(ultima_hsamp_linear_args)); return 0; }\n'
    with tempfile.TemporaryDirectory() as d:
        (Path(d) / "s.c").write_text(src)
        subprocess.run(["gcc", f"-I{hsamp.HEADER.parent}", "-o", f"{d}/s", f"{d}/s.c"], check=True)
        sizes = subprocess.run([f"{d}/s"], capture_output=True, text=True, check=True).stdout.split()
    assert [int(s) for s in sizes] == [ctypes.sizeof(c) for c in (hsamp.Draft, hsamp.DraftSets, hsamp.LinearArgs)]
