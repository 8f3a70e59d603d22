"""What quantize_rows, linear_i8, cross_entropy(_grad), embed and embed_grad refuse,
without a GPU: every call here returns before anything is launched."""
import ctypes

import pytest

OK_PTR = 1 << 20      # never looked at: the call is refused first


@pytest.fixture(scope="module")
def hsamp(pkg):
    return pkg.hsamp


def call(hsamp, struct, name, fields, kw):
    a = struct()
    for k, v in {**fields, **kw}.items():
        setattr(a, k, v)
    return getattr(hsamp.lib(), f"ultima_hsamp_{name}")(ctypes.byref(a), None)


LINEAR = dict(rows=4, in_dim=32, out_dim=16, groups=1, dtype=1, out_dtype=1, act=0, x=OK_PTR, x_stride=32, x_scale=OK_PTR + 64,
              weight=2 * OK_PTR, weight_stride=32, weight_scale=OK_PTR + 128, out=3 * OK_PTR, out_stride=16)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(rows=-1), dict(in_dim=0), dict(out_dim=0), dict(groups=0), dict(dtype=0), dict(dtype=2), dict(out_dtype=9),
    dict(act=-1), dict(act=6), dict(act=5, act_param=0.0), dict(act=5, act_param=-1.0), dict(act=5, act_param=float("inf")),
    dict(act=5, act_param=float("nan")), dict(x=None), dict(x_scale=None), dict(weight=None), dict(weight_scale=None), dict(out=None),
    dict(x_stride=31), dict(weight_stride=31), dict(out_stride=15), dict(residual=OK_PTR, residual_stride=15), dict(x_scale=OK_PTR + 2),
    dict(weight_scale=OK_PTR + 1), dict(out=3 * OK_PTR + 1), dict(out_dtype=0, out=3 * OK_PTR + 2), dict(bias=OK_PTR + 1),
    dict(out=OK_PTR), dict(out=2 * OK_PTR), dict(out=OK_PTR + 64), dict(out=OK_PTR + 128),
    dict(out_dtype=0, residual=3 * OK_PTR, residual_stride=16), dict(residual=3 * OK_PTR, residual_stride=17),
    dict(groups=2, out_group=0), dict(groups=2, out_group=15), dict(groups=2, out_group=63),
])
def test_linear_i8_refuses(hsamp, kw):
    assert call(hsamp, hsamp.LinearI8Args, "linear_i8", LINEAR, kw) == hsamp.ERR_INVALID


def test_linear_i8_refuses_null_and_too_much(hsamp):
    assert hsamp.lib().ultima_hsamp_linear_i8(None, None) == hsamp.ERR_INVALID
    for kw in (dict(in_dim=131072, x_stride=131072, weight_stride=131072), dict(groups=65536, out_group=64),
               dict(rows=1 << 30, out_dim=1 << 20, out_stride=1 << 20)):
        assert call(hsamp, hsamp.LinearI8Args, "linear_i8", LINEAR, kw) == hsamp.ERR_UNSUPPORTED


QUANTIZE = dict(rows=4, in_dim=32, dtype=1, x=OK_PTR, x_stride=32, q=2 * OK_PTR, q_stride=32, scale=3 * OK_PTR)


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(in_dim=0), dict(dtype=2), dict(dtype=-1), dict(x=None), dict(q=None), dict(scale=None), dict(x_stride=31),
    dict(q_stride=31), dict(x=OK_PTR + 1), dict(dtype=0, x=OK_PTR + 2), dict(scale=3 * OK_PTR + 2), dict(q=OK_PTR), dict(scale=OK_PTR),
])
def test_quantize_rows_refuses(hsamp, kw):
    assert call(hsamp, hsamp.QuantizeArgs, "quantize_rows", QUANTIZE, kw) == hsamp.ERR_INVALID


def test_quantize_rows_refuses_null_and_too_much(hsamp):
    assert hsamp.lib().ultima_hsamp_quantize_rows(None, None) == hsamp.ERR_INVALID
    assert call(hsamp, hsamp.QuantizeArgs, "quantize_rows", QUANTIZE, dict(rows=1 << 24)) == hsamp.ERR_UNSUPPORTED


LOSS = dict(rows=4, in_dim=32, vocab=100, dtype=1, x=OK_PTR, x_stride=32, weight=2 * OK_PTR, weight_stride=32, target=3 * OK_PTR,
            lse=4 * OK_PTR, work=5 * OK_PTR)
FORWARD = dict(LOSS, loss=6 * OK_PTR)
GRAD = dict(LOSS, grad=6 * OK_PTR, d_x=7 * OK_PTR, d_x_stride=32, d_x_dtype=1, d_weight=8 * OK_PTR, d_weight_stride=32, d_weight_dtype=0)
EITHER = [
    dict(rows=0), dict(rows=-5), dict(in_dim=0), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(dtype=0), dict(dtype=2), dict(softcap=-1.0),
    dict(softcap=float("inf")), dict(softcap=float("nan")), dict(x=None), dict(weight=None), dict(target=None), dict(lse=None),
    dict(work=None), dict(x_stride=31), dict(weight_stride=31), dict(x=OK_PTR + 1), dict(weight=OK_PTR + 1), dict(target=OK_PTR + 2),
    dict(lse=OK_PTR + 1), dict(work=OK_PTR + 8),
]


@pytest.mark.parametrize("kw", EITHER + [dict(loss=None), dict(loss=OK_PTR + 2), dict(loss=4 * OK_PTR)])
def test_cross_entropy_refuses(hsamp, kw):
    assert call(hsamp, hsamp.CrossEntropyArgs, "cross_entropy", FORWARD, kw) == hsamp.ERR_INVALID


@pytest.mark.parametrize("kw", EITHER + [
    dict(grad=None), dict(grad=OK_PTR + 2), dict(d_x=None, d_weight=None), dict(d_x_stride=31), dict(d_weight_stride=31), dict(d_x_dtype=9),
    dict(d_weight_dtype=9), dict(d_x=OK_PTR + 1), dict(d_weight=OK_PTR + 2), dict(d_x=OK_PTR), dict(d_weight=2 * OK_PTR),
    dict(d_weight=7 * OK_PTR), dict(d_x=5 * OK_PTR), dict(d_x=4 * OK_PTR), dict(d_weight=6 * OK_PTR), dict(d_x=3 * OK_PTR),
])
def test_cross_entropy_grad_refuses(hsamp, kw):
    assert call(hsamp, hsamp.CrossEntropyGradArgs, "cross_entropy_grad", GRAD, kw) == hsamp.ERR_INVALID


def test_cross_entropy_refuses_null_and_too_much(hsamp):
    L = hsamp.lib()
    assert L.ultima_hsamp_cross_entropy(None, None) == L.ultima_hsamp_cross_entropy_grad(None, None) == hsamp.ERR_INVALID
    for struct, name, fields in ((hsamp.CrossEntropyArgs, "cross_entropy", FORWARD), (hsamp.CrossEntropyGradArgs, "cross_entropy_grad", GRAD)):
        for kw in (dict(rows=(1 << 22) + 1), dict(rows=1 << 22, in_dim=1024, x_stride=1024, weight_stride=1024, d_x_stride=1024, d_weight_stride=1024),
                   dict(rows=1 << 22, vocab=1 << 24)):
            assert call(hsamp, struct, name, fields, {k: v for k, v in kw.items() if hasattr(struct, k)}) == hsamp.ERR_UNSUPPORTED


def test_cross_entropy_work_bytes(hsamp):
    f, g = hsamp.lib().ultima_hsamp_cross_entropy_work_bytes, hsamp.lib().ultima_hsamp_cross_entropy_grad_work_bytes
    assert f(0, 5) == -1 and f(5, 0) == -1 and f(1, (1 << 24) + 1) == -1
    assert g(0, 5, 5) == -1 and g(5, 0, 5) == -1 and g(5, 5, 0) == -1 and g(1, 1, (1 << 24) + 1) == -1
    assert 0 < f(1, 1) <= f(2, 1) <= f(2, 151936) and f(1 << 22, 1 << 24) > 2**40
    # a piece of the vocabulary at a time: not the logits
    assert g(4096, 4096, 151936) < 1 << 29 and g(4096, 4096, 1 << 24) < 1 << 29


EMBED = dict(tokens=4, width=32, vocab=100, dtype=1, out_dtype=1, scale=1.0, table=OK_PTR, table_stride=32, ids=2 * OK_PTR, out=3 * OK_PTR,
             out_stride=32)
EMBED_GRAD = dict(tokens=4, width=32, vocab=100, dtype=1, out_dtype=1, scale=1.0, d_out=OK_PTR, d_out_stride=32, ids=2 * OK_PTR,
                  out=3 * OK_PTR, out_stride=32, work=4 * OK_PTR)
ROWS = [
    dict(tokens=0), dict(tokens=-1), dict(width=0), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(dtype=2), dict(out_dtype=9), dict(dtype=0),
    dict(ids=None), dict(out=None), dict(out_stride=31), dict(out=3 * OK_PTR + 1), dict(out_dtype=0, out=3 * OK_PTR + 2), dict(ids=OK_PTR + 2),
    dict(out=OK_PTR), dict(out=2 * OK_PTR),
]


@pytest.mark.parametrize("kw", ROWS + [dict(table=None), dict(table_stride=31), dict(table=OK_PTR + 1), dict(dtype=0, out_dtype=0, table=OK_PTR + 2)])
def test_embed_refuses(hsamp, kw):
    assert call(hsamp, hsamp.EmbedArgs, "embed", EMBED, kw) == hsamp.ERR_INVALID


@pytest.mark.parametrize("kw", ROWS + [dict(d_out=None), dict(d_out_stride=31), dict(d_out=OK_PTR + 1), dict(work=None), dict(work=OK_PTR + 8),
                                       dict(out=4 * OK_PTR)])
def test_embed_grad_refuses(hsamp, kw):
    assert call(hsamp, hsamp.EmbedGradArgs, "embed_grad", EMBED_GRAD, kw) == hsamp.ERR_INVALID


def test_embed_refuses_null_and_too_much(hsamp):
    L = hsamp.lib()
    assert L.ultima_hsamp_embed(None, None) == L.ultima_hsamp_embed_grad(None, None) == hsamp.ERR_INVALID
    big = dict(width=(1 << 24) + 1, table_stride=1 << 25, d_out_stride=1 << 25, out_stride=1 << 25)
    for struct, name, fields in ((hsamp.EmbedArgs, "embed", EMBED), (hsamp.EmbedGradArgs, "embed_grad", EMBED_GRAD)):
        for kw in (big, dict(tokens=(1 << 30) + 1), dict(tokens=1 << 30)):
            assert call(hsamp, struct, name, fields, {k: v for k, v in kw.items() if hasattr(struct, k)}) == hsamp.ERR_UNSUPPORTED


def test_embed_grad_work_bytes(hsamp):
    f = hsamp.lib().ultima_hsamp_embed_grad_work_bytes
    assert f(0, 5, 5) == -1 and f(5, 0, 5) == -1 and f(5, 5, 0) == -1 and f(1, 1, (1 << 24) + 1) == -1
    assert 0 < f(1, 1, 1) <= f(64, 1, 1) <= f(64, 100, 1) <= f(64, 100, 1000)


def test_struct_layouts_match_the_header(hsamp, tmp_path):
    import subprocess
    structs = {"linear_i8_args": hsamp.LinearI8Args, "quantize_args": hsamp.QuantizeArgs, "cross_entropy_args": hsamp.CrossEntropyArgs,
               "cross_entropy_grad_args": hsamp.CrossEntropyGradArgs, "embed_args": hsamp.EmbedArgs, "embed_grad_args": hsamp.EmbedGradArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ultima_hsamp.h"', 'int main(void) {']
    want = []
    for name, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof(ultima_hsamp_{name}));')
        want.append(ctypes.sizeof(py))
        for field, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof(ultima_hsamp_{name}, {field}));')
            want.append(getattr(py, field).offset)
    (tmp_path / "t.c").write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-std=c11", f"-I{hsamp.HEADER.parent}", str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout
    assert [int(v) for v in out.split()] == want


def test_tensors_on_the_host_are_refused(hsamp):
    import torch
    b, q, i = torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros((2, 8), dtype=torch.int8), torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2)
    for fn, args in ((hsamp.quantize_rows, (b,)), (hsamp.linear_i8, (q, f, q, f)), (hsamp.cross_entropy, (b, b, i)),
                     (hsamp.cross_entropy_grad, (b, b, i, f, f)), (hsamp.embed, (b, i)), (hsamp.embed_grad, (b, i, 5))):
        with pytest.raises(hsamp.HsampError) as e:
            fn(*args)
        assert e.value.status == hsamp.ERR_INVALID
