"""Refusals of token_logprobs and topk_distillation_loss without a GPU: the C entry points check their
arguments on the host before they touch a device, and the Python functions check tensors (fake ones
on a CUDA device here, which hold shapes and types but no data) before they call the library."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses import FakeTensorMode

from macrogpt_jax_b200 import _capi as C

P = 1 << 20  # stands for a 16-byte aligned device address; no call here reads it


def rows(**kw):
    a = dict(ptr=P, dtype=C.OUT_BF16, temperature=1.0, rows=4, V=100, inner=4, stride_outer=0, stride_inner=100,
             mask=None)
    a.update(kw)
    return C.LogitRows(*(a[f] for f, _ in C.LogitRows._fields_))


def fwd(r, tokens=P, token_bytes=8, k=0, lp=P, ent=P, top=None, ids=None, stats=None):
    return C.load().ufp8_logprob_forward(None if r is None else ctypes.byref(r), tokens, token_bytes, k, lp, ent, top,
                                         ids, stats, None)


def bwd(r, stats=P, tokens=P, token_bytes=8, dlp=P, dtop=None, ids=None, k=0, cap=0.0, fmt=C.LIKE_LOGITS, out=P,
        outer=400, inner=100, amax=None, inv=None):
    return C.load().ufp8_logprob_backward(ctypes.byref(r), stats, tokens, token_bytes, dlp, 1, None, 0, dtop, ids, k,
                                          cap, fmt, out, outer, inner, amax, inv, None)


def dfwd(r, ids=P, id_bytes=8, teacher=P, dtype=C.OUT_F32, k=4, loss=P, stats=None):
    return C.load().ufp8_distill_forward(ctypes.byref(r), ids, id_bytes, teacher, dtype, k, loss, stats, None)


def dbwd(r, stats=P, ids=P, id_bytes=8, teacher=P, dtype=C.OUT_F32, k=4, dloss=P, cap=0.0, fmt=C.LIKE_LOGITS,
         out=P, outer=400, inner=100, amax=None, inv=None):
    return C.load().ufp8_distill_backward(ctypes.byref(r), stats, ids, id_bytes, teacher, dtype, k, dloss, 1, cap,
                                          fmt, out, outer, inner, amax, inv, None)


@pytest.mark.parametrize("call,code,msg", [
    (lambda: fwd(None), C.ERR_INVALID, "null rows"),
    (lambda: fwd(rows(dtype=7)), C.ERR_INVALID, "dtype 7"),
    (lambda: fwd(rows(rows=-1)), C.ERR_INVALID, "rows must be >= 0"),
    (lambda: fwd(rows(V=0)), C.ERR_INVALID, "V >= 1"),
    (lambda: fwd(rows(V=1 << 31)), C.ERR_INVALID, "V exceeds"),
    (lambda: fwd(rows(rows=1 << 31)), C.ERR_INVALID, "rows exceed"),
    (lambda: fwd(rows(inner=0)), C.ERR_INVALID, "inner"),
    (lambda: fwd(rows(temperature=0.0)), C.ERR_INVALID, "temperature"),
    (lambda: fwd(rows(temperature=float("inf"))), C.ERR_INVALID, "temperature"),
    (lambda: fwd(rows(temperature=float("nan"))), C.ERR_INVALID, "temperature"),
    (lambda: fwd(rows(temperature=1e-35)), C.ERR_INVALID, "out of range"),
    (lambda: fwd(rows(ptr=None)), C.ERR_INVALID, "null logits"),
    (lambda: fwd(rows(ptr=P + 1)), C.ERR_ALIGN, "logits not aligned"),
    (lambda: fwd(rows(ptr=P + 2, dtype=C.OUT_F32)), C.ERR_ALIGN, "logits not aligned"),
    (lambda: fwd(rows(), token_bytes=2), C.ERR_INVALID, "tokens of 2 bytes"),
    (lambda: fwd(rows(), tokens=P + 4), C.ERR_ALIGN, "tokens not aligned"),
    (lambda: fwd(rows(), tokens=None), C.ERR_INVALID, "go together"),
    (lambda: fwd(rows(), lp=None), C.ERR_INVALID, "go together"),
    (lambda: fwd(rows(), tokens=None, lp=None, ent=None), C.ERR_INVALID, "no output"),
    (lambda: fwd(rows(), k=257, top=P, ids=P), C.ERR_INVALID, "top_k must be"),
    (lambda: fwd(rows(), k=101, top=P, ids=P), C.ERR_INVALID, "top_k exceeds V"),
    (lambda: fwd(rows(), k=3, top=P), C.ERR_INVALID, "null top"),
    (lambda: fwd(rows(), stats=P + 8), C.ERR_ALIGN, "stats"),
    (lambda: bwd(rows(), stats=None), C.ERR_INVALID, "null stats"),
    (lambda: bwd(rows(), out=None), C.ERR_INVALID, "null stats or dlogits"),
    (lambda: bwd(rows(), out=P + 1), C.ERR_ALIGN, "dlogits not aligned"),
    (lambda: bwd(rows(), inner=99), C.ERR_INVALID, "overlap"),
    (lambda: bwd(rows(inner=2), outer=199), C.ERR_INVALID, "overlap"),
    (lambda: bwd(rows(), tokens=None), C.ERR_INVALID, "null tokens"),
    (lambda: bwd(rows(), dtop=P, k=3), C.ERR_INVALID, "null top_ids"),
    (lambda: bwd(rows(), dtop=P, ids=P, k=0), C.ERR_INVALID, "null top_ids"),
    (lambda: bwd(rows(), cap=-1.0), C.ERR_INVALID, "cap must be"),
    (lambda: bwd(rows(), cap=float("inf")), C.ERR_INVALID, "cap must be"),
    (lambda: dbwd(rows(), cap=float("nan")), C.ERR_INVALID, "cap must be"),
    (lambda: bwd(rows(), cap=15.0), C.ERR_UNSUPPORTED, "cap needs fp8"),
    (lambda: bwd(rows(), fmt=C.BF16), C.ERR_INVALID, "fmt 2"),
    (lambda: bwd(rows(dtype=C.OUT_F32), fmt=C.E5M2, amax=P, inv=P), C.ERR_UNSUPPORTED, "bf16"),
    (lambda: dbwd(rows(dtype=C.OUT_F32), fmt=C.E4M3, amax=P, inv=P), C.ERR_UNSUPPORTED, "bf16"),
    (lambda: bwd(rows(), fmt=C.E5M2), C.ERR_INVALID, "null amax"),
    (lambda: dbwd(rows(), fmt=C.E5M2, amax=P), C.ERR_INVALID, "null amax or inv_scale"),
    (lambda: bwd(rows(), fmt=C.E5M2, amax=P + 2, inv=P), C.ERR_ALIGN, "amax"),
    (lambda: dfwd(rows(), k=-1), C.ERR_INVALID, "entries must be"),
    (lambda: dfwd(rows(), k=1025), C.ERR_INVALID, "entries must be"),
    (lambda: dfwd(rows(), dtype=9), C.ERR_INVALID, "teacher_dtype 9"),
    (lambda: dfwd(rows(), id_bytes=1), C.ERR_INVALID, "teacher ids of 1"),
    (lambda: dfwd(rows(), ids=None), C.ERR_INVALID, "null teacher"),
    (lambda: dfwd(rows(), teacher=P + 2), C.ERR_ALIGN, "teacher not aligned"),
    (lambda: dfwd(rows(), loss=None), C.ERR_INVALID, "null loss"),
    (lambda: dbwd(rows(), dloss=None), C.ERR_INVALID, "null stats, dloss"),
    (lambda: dbwd(rows(), inner=50), C.ERR_INVALID, "overlap"),
])
def test_entry_points_refuse(call, code, msg):
    assert call() == code
    assert msg in C.load().ufp8_last_error().decode()


def test_no_rows_is_no_launch():
    """Zero rows: every entry point returns before it looks for a device."""
    r = rows(rows=0, ptr=None, inner=1)
    assert fwd(r) == C.OK and bwd(r) == C.OK and dfwd(r) == C.OK and dbwd(r) == C.OK


def test_struct_layout(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    prints = "".join(f'printf("%zu\\n", offsetof(ufp8_logit_rows, {f}));' for f, _ in C.LogitRows._fields_)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ufp8.h"\nint main(void) {'
                   'printf("%zu\\n", sizeof(ufp8_logit_rows));' + prints + "return 0; }")
    subprocess.run([cc, "-I", str(Path(__file__).resolve().parents[1] / "include"), str(src), "-o",
                    str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                          text=True).stdout.split()]
    assert got == [ctypes.sizeof(C.LogitRows)] + [getattr(C.LogitRows, f).offset for f, _ in C.LogitRows._fields_]


def _score(**kw):
    from macrogpt_jax_b200.logprobs import token_logprobs
    return token_logprobs(**kw)


def _distill(**kw):
    from macrogpt_jax_b200.distill import topk_distillation_loss
    return topk_distillation_loss(**kw)


@pytest.mark.parametrize("make,error,match", [
    (lambda e: _score(logits=e(2, 8, device="cpu"), tokens=e(2, dtype=torch.int64)), ValueError, "CUDA"),
    (lambda e: _score(logits=e(2, 8, dtype=torch.float16), tokens=e(2, dtype=torch.int64)), TypeError, "float16"),
    (lambda e: _score(logits=e(2, 0)), ValueError, "no columns"),
    (lambda e: _score(logits=e(2, 8), tokens=e(3, dtype=torch.int64)), ValueError, "tokens"),
    (lambda e: _score(logits=e(2, 8), tokens=e(2, dtype=torch.int64, device="cpu")), ValueError, "tokens"),
    (lambda e: _score(logits=e(2, 8), tokens=e(2)), TypeError, "integers"),
    (lambda e: _score(logits=e(2, 8), tokens=e(2, dtype=torch.bool)), TypeError, "integers"),
    (lambda e: _score(logits=e(2, 8), top_k=9), ValueError, "top_k"),
    (lambda e: _score(logits=e(2, 800), top_k=257), ValueError, "top_k"),
    (lambda e: _score(logits=e(2, 8), top_k=-1), ValueError, "top_k"),
    (lambda e: _score(logits=e(2, 8), entropy=False), ValueError, "nothing asked"),
    (lambda e: _score(logits=e(2, 8), temperature=0.0), ValueError, "temperature"),
    (lambda e: _score(logits=e(2, 8), temperature=float("nan")), ValueError, "temperature"),
    (lambda e: _score(logits=e(2, 8), mask=e(8, dtype=torch.bool)), ValueError, "mask"),
    (lambda e: _score(logits=e(2, 8), mask=e(2)), TypeError, "mask"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 3, dtype=torch.int64), teacher_logits=e(2, 4)), ValueError,
     "teacher_logits"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(3, 3, dtype=torch.int64), teacher_logits=e(3, 3)), ValueError,
     "teacher_ids"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 1025, dtype=torch.int64), teacher_logits=e(2, 1025)),
     ValueError, "1024"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 3), teacher_logits=e(2, 3)), TypeError, "integers"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 3, dtype=torch.int64),
                        teacher_logits=e(2, 3, dtype=torch.float64)), TypeError, "float64"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 3, dtype=torch.int64),
                        teacher_logits=e(2, 3).requires_grad_(True)), ValueError, "no gradient"),
    (lambda e: _distill(logits=e(2, 8), teacher_ids=e(2, 3, dtype=torch.int64), teacher_logits=e(2, 3),
                        temperature=-1.0), ValueError, "temperature"),
])
def test_functions_refuse(make, error, match):
    with FakeTensorMode():
        def empty(*shape, **kw):
            return torch.empty(shape, **{"device": "cuda", **kw})
        with pytest.raises(error, match=match):
            make(empty)


@pytest.mark.parametrize("shape,strides,start,expect", [
    # (tensor shape, strides, offset in a buffer) -> (rows, inner, stride_outer, stride_inner)
    ((3, 5, 16), (80, 16, 1), 0, (15, 15, 0, 16)),
    ((3, 4, 17), (85, 17, 1), 0, (12, 4, 85, 17)),       # logits[:, :-1]
    ((3, 5, 17), (120, 24, 1), 0, (15, 15, 0, 24)),      # padded columns
    ((7,), (1,), 3, (1, 1, 0, 7)),
    ((2, 1, 5), (50, 7, 1), 0, (2, 2, 0, 50)),
    ((4, 6), (0, 1), 0, (4, 4, 0, 0)),                   # one row expanded
    ((2, 3, 4, 5), (120, 20, 5, 1), 0, (24, 12, 120, 5)),
])
def test_row_views(shape, strides, start, expect):
    """Rows are addressed in place for up to two levels of strides, and the gradient's rows start as
    far from a 16-byte boundary as the logit rows without overlapping."""
    from macrogpt_jax_b200 import ops
    buf = torch.arange(4096, dtype=torch.float32)
    t = buf.as_strided(shape, strides, start)
    lr = ops.logit_rows(t)
    assert lr.logits is t
    assert (lr.rows, lr.inner, lr.stride_outer, lr.stride_inner) == expect
    flat = t.reshape(-1, shape[-1])
    for r in range(lr.rows):
        e = start + (r // lr.inner) * lr.stride_outer + (r % lr.inner) * lr.stride_inner
        assert torch.equal(flat[r], buf[e:e + shape[-1]])
    g, outer, inner = ops._grad_rows(lr)
    assert g.shape == t.shape
    seen = set()
    for r in range(lr.rows):
        e = (r // lr.inner) * outer + (r % lr.inner) * inner
        src = t.data_ptr() + 4 * ((r // lr.inner) * lr.stride_outer + (r % lr.inner) * lr.stride_inner)
        assert (g.data_ptr() + 4 * e - src) % 16 == 0
        cols = set(range(e, e + shape[-1]))
        assert not cols & seen
        seen |= cols


def test_three_stride_levels_are_copied():
    from macrogpt_jax_b200 import ops
    t = torch.arange(2 * 3 * 4 * 8, dtype=torch.float32).reshape(2, 3, 4, 8)[:, :2, :3]
    lr = ops.logit_rows(t)
    assert lr.logits.is_contiguous() and torch.equal(lr.logits, t) and lr.rows == 12
