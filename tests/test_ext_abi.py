"""CPU: the entry points of include/kernel_set/ext are exported, bound and refuse what they do not take."""
import ctypes
import glob
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p
ONE, TWO, ODD = P(16), P(32), P(50)   # tokens for addresses; argument checks never dereference them
F, I = ctypes.POINTER(ctypes.c_float), ctypes.POINTER(ctypes.c_int32)


def f32p(v):
    return ctypes.cast(v, F)


def i32p(v):
    return ctypes.cast(v, I)


def test_declared_and_exported(ks):
    names = []
    for h in sorted(glob.glob(os.path.join(ROOT, "include", "kernel_set", "ext", "*.h"))):
        text = re.sub(r"/\*.*?\*/", "", open(h).read(), flags=re.S)
        names += re.findall(r"KS_API[^;(]*?\b(ks_[a-z0-9_]+)\s*\(", text)
    assert len(names) == len(set(names)) == 7
    out = subprocess.run(["nm", "-D", "--defined-only", ks.LIB_PATH], capture_output=True, text=True, check=True)
    exported = {l.split()[-1] for l in out.stdout.splitlines() if " T " in l}
    assert set(names) <= exported
    assert all(getattr(ks._lib.lib, n).argtypes is not None for n in names)


def test_moe_backward_refusals(ks):
    L, S, D = ks._lib.lib, ks.Status, ks.DType
    up = lambda dp=ONE, dw=ONE, do=TWO, p=ONE, ids=ONE, w=ONE, t=4, k=2, h=8, dt=D.BF16: L.ks_moe_unpermute_backward(  # noqa: E731
        dp, f32p(dw), do, p, i32p(ids), f32p(w), t, k, h, dt, None)
    for bad in (dict(dp=None), dict(dw=P()), dict(do=None), dict(p=None), dict(ids=P()), dict(w=P()), dict(t=-1), dict(k=0), dict(h=0),
                dict(dp=TWO)):
        assert up(**bad) == S.INVALID_ARGUMENT, bad
    assert up(dt=D.I8) == S.UNSUPPORTED_DTYPE and up(dt=D.F8E4M3) == S.UNSUPPORTED_DTYPE
    assert up(t=2 ** 31) == S.UNSUPPORTED_SHAPE
    assert up(t=2 ** 30 - 1) == S.UNSUPPORTED_SHAPE      # the grid
    assert up(t=0, dp=None, p=None) == S.SUCCESS
    pb = lambda di=ONE, dp=TWO, ids=ONE, t=4, k=2, h=8, dt=D.BF16: L.ks_moe_permute_backward(  # noqa: E731
        di, dp, i32p(ids), t, k, h, dt, None)
    for bad in (dict(di=None), dict(dp=None), dict(ids=P()), dict(t=-1), dict(k=0), dict(h=0), dict(dp=ONE)):
        assert pb(**bad) == S.INVALID_ARGUMENT, bad
    assert pb(dt=D.F8E5M2) == S.UNSUPPORTED_DTYPE
    assert pb(t=2 ** 31) == S.UNSUPPORTED_SHAPE and pb(k=5000) == S.UNSUPPORTED_SHAPE
    assert pb(t=0, di=None, dp=None) == S.SUCCESS
    gb = lambda dl=ONE, dw=ONE, w=ONE, i=ONE, l=TWO, t=4, e=8, k=2, rn=0, dt=D.F32: L.ks_moe_gate_softmax_topk_backward(  # noqa: E731
        dl, f32p(dw), f32p(w), i32p(i), l, t, e, k, rn, dt, None)
    for bad in (dict(dl=None), dict(dw=P()), dict(w=P()), dict(i=P()), dict(l=None), dict(t=-1), dict(e=0), dict(k=0), dict(k=9)):
        assert gb(**bad) == S.INVALID_ARGUMENT, bad
    assert gb(e=1025, k=2) == S.UNSUPPORTED_SHAPE and gb(e=64, k=33) == S.UNSUPPORTED_SHAPE
    assert gb(dt=D.I8) == S.UNSUPPORTED_DTYPE
    assert gb(t=0, dl=None, l=None) == S.SUCCESS


def test_lora_refusals(ks):
    L, S, D = ks._lib.lib, ks.Status, ks.DType

    def ap(out=ONE, ldo=32, base=ONE, ldb=32, h=P(), x=TWO, ldx=64, a=ONE, b=ONE, s=ONE, ids=ONE, off=ONE, t=4, l=2, r=8, k=64, n=32,
           dt=D.BF16):
        return L.ks_lora_apply(out, ldo, base, ldb, f32p(h), x, ldx, a, b, f32p(s), i32p(ids), i32p(off), t, l, r, k, n, dt, None)

    for bad in (dict(out=None), dict(base=None), dict(x=None), dict(a=None), dict(b=None), dict(s=P()), dict(off=P()), dict(t=-1),
                dict(l=0), dict(r=0), dict(k=0), dict(n=0), dict(ldx=63), dict(ldo=31), dict(ldb=31), dict(ldo=40), dict(x=ONE)):
        assert ap(**bad) == S.INVALID_ARGUMENT, bad
    for dt in (D.F32, D.F8E4M3, D.I8):
        assert ap(dt=dt) == S.UNSUPPORTED_DTYPE
    for bad in (dict(l=1024), dict(r=4097), dict(t=2 ** 31), dict(k=2 ** 30, ldx=2 ** 30), dict(n=2 ** 30, ldo=2 ** 30, ldb=2 ** 30)):
        assert ap(**bad) == S.UNSUPPORTED_SHAPE, bad
    assert ap(t=0, out=None, base=None, x=None) == S.SUCCESS

    def bw(dx=ONE, lddx=64, da=ONE, db=ONE, dxb=ONE, lddxb=64, do=TWO, lddo=32, x=TWO, ldx=64, h=ONE, a=ONE, b=ONE, s=ONE, ids=ONE,
           off=ONE, t=4, l=2, r=8, k=64, n=32, ws=ONE, wsb=1 << 20, dt=D.BF16):
        return L.ks_lora_backward(dx, lddx, da, db, dxb, lddxb, do, lddo, x, ldx, f32p(h), a, b, f32p(s), i32p(ids), i32p(off), t, l, r,
                                  k, n, ws, wsb, dt, None)

    for bad in (dict(dx=None), dict(da=None), dict(db=None), dict(dxb=None), dict(do=None), dict(x=None), dict(h=P()), dict(a=None),
                dict(b=None), dict(s=P()), dict(off=P()), dict(t=-1), dict(l=0), dict(lddx=63), dict(lddo=31), dict(ldx=63), dict(lddxb=63),
                dict(lddx=72), dict(do=ONE), dict(x=ONE), dict(ws=None), dict(ws=ODD), dict(wsb=16)):
        assert bw(**bad) == S.INVALID_ARGUMENT, bad
    assert bw(dt=D.F32) == S.UNSUPPORTED_DTYPE
    assert bw(l=1024) == S.UNSUPPORTED_SHAPE
    size = ctypes.c_size_t()
    assert L.ks_lora_backward_workspace(None, 4, 2, 8, 64, 32) == S.INVALID_ARGUMENT
    assert L.ks_lora_backward_workspace(ctypes.byref(size), 4, 0, 8, 64, 32) == S.INVALID_ARGUMENT
    assert L.ks_lora_backward_workspace(ctypes.byref(size), 1000, 2, 8, 64, 32) == S.SUCCESS and size.value >= 1000 * 8 * 4
    assert L.ks_lora_plan(i32p(ONE), i32p(P()), i32p(ONE), 4, 2, None) == S.INVALID_ARGUMENT
    assert L.ks_lora_plan(i32p(P()), i32p(ONE), i32p(ONE), 4, 2, None) == S.INVALID_ARGUMENT
    assert L.ks_lora_plan(i32p(ONE), i32p(ONE), i32p(ONE), 4, 0, None) == S.INVALID_ARGUMENT
    assert L.ks_lora_plan(i32p(ONE), i32p(ONE), i32p(ONE), 4, 1024, None) == S.UNSUPPORTED_SHAPE


def test_python_wrappers_refuse(ks):
    bf = torch.bfloat16
    a, b, s = torch.zeros(2, 8, 64, dtype=bf), torch.zeros(2, 32, 8, dtype=bf), torch.zeros(2)
    x, y, off, ids = torch.zeros(4, 64, dtype=bf), torch.zeros(4, 32, dtype=bf), torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    call = lambda **v: ks.lora.apply(*[{**dict(out=y, base=y, x=x, a=a, b=b, scales=s, sorted_ids=ids, offsets=off), **v}[n]  # noqa: E731
                                       for n in ("out", "base", "x", "a", "b", "scales", "sorted_ids", "offsets")], **{
                                           n: v[n] for n in ("h",) if n in v})
    with pytest.raises(ValueError, match="CUDA tensor"):
        call()
    for bad, what in ((dict(b=torch.zeros(2, 32, 16, dtype=bf)), "b"), (dict(scales=torch.zeros(3)), "scales"), (dict(offsets=off[:2]), "offsets"),
                      (dict(sorted_ids=ids[:3]), "sorted_ids"), (dict(sorted_ids=ids.long()), "int32"), (dict(scales=s.double()), "float32"),
                      (dict(a=a.half()), "bfloat16"), (dict(out=y.float()), "bfloat16"), (dict(x=x[0]), "x must be")):
        with pytest.raises(ValueError, match=what):
            call(**bad)
    with pytest.raises(ValueError, match="int32"):
        ks.lora.plan(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="must be"):
        ks.moe.permute_backward(torch.zeros(2, 8), torch.zeros(4, 8, dtype=bf), ids, 2, 2, 8)


def test_moe_backward_wrappers_refuse(ks):
    """Types and sizes that would be read as something else, or beyond the end (torch.topk's indices are 64-bit, for one)."""
    f, i = torch.zeros(4, 2), torch.zeros(8, dtype=torch.int32)
    rows, pairs = torch.zeros(4, 8), torch.zeros(8, 8)
    up = dict(d_permuted=pairs, d_weights=f, d_out=rows, permuted=pairs, sorted_token_ids=i, routing_weights=f, num_tokens=4, top_k=2, hidden=8)
    pb = dict(d_input=rows, d_permuted=pairs, sorted_token_ids=i, num_tokens=4, top_k=2, hidden=8)
    gb = dict(d_logits=rows, d_weights=f, weights=f, indices=i, logits=rows, num_tokens=4, num_experts=8, top_k=2)
    for fn, good, bad in ((ks.moe.unpermute_backward, up, (dict(d_weights=f.half()), dict(routing_weights=f[:3]), dict(sorted_token_ids=i.long()),
                                                           dict(permuted=pairs[:7]), dict(d_out=rows[:3]), dict(d_permuted=pairs.half()))),
                          (ks.moe.permute_backward, pb, (dict(sorted_token_ids=i[:7]), dict(d_permuted=pairs[:7]), dict(d_input=rows[:3]))),
                          (ks.moe.gate_softmax_topk_backward, gb, (dict(indices=i.long()), dict(weights=f.double()), dict(d_weights=f[:3]),
                                                                   dict(logits=rows[:3]), dict(d_logits=rows.half())))):
        with pytest.raises(ValueError, match="CUDA tensor"):
            fn(**good)
        for b in bad:
            with pytest.raises(ValueError, match="must be torch|elements where"):
                fn(**{**good, **b})


def test_plan_refuses_buffers_of_other_types_and_sizes(ks):
    """They are written as int32: 64-bit ones have the right count and would hold pairs of numbers."""
    ids = torch.zeros(6, dtype=torch.int32)
    for sorted_ids, offsets, what in ((torch.zeros(6, dtype=torch.int64), None, "sorted_ids must be int32"),
                                      (None, torch.zeros(4, dtype=torch.int64), "offsets must be int32"),
                                      (torch.zeros(6), None, "sorted_ids must be int32"),
                                      (torch.zeros(5, dtype=torch.int32), None, "expected"),
                                      (None, torch.zeros(5, dtype=torch.int32), "expected")):
        with pytest.raises(ValueError, match=what):
            ks.lora.plan(ids, 2, sorted_ids, offsets)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ks.lora.plan(ids, 2, torch.zeros(6, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


def test_moe_backward_wrappers_refuse_a_dtype_that_is_not_the_tensors(ks):
    """A given dtype is for raw addresses; one wider than the tensors' would be read beyond their ends."""
    bf, f, i = torch.bfloat16, torch.zeros(4, 2), torch.zeros(8, dtype=torch.int32)
    rows, pairs = torch.zeros(4, 8, dtype=bf), torch.zeros(8, 8, dtype=bf)
    for dtype, match in ((ks.DType.F32, "as dtype says"), (ks.DType.F16, "as dtype says"), (ks.DType.BF16, "CUDA tensor")):
        with pytest.raises(ValueError, match=match):
            ks.moe.unpermute_backward(pairs, f, rows, pairs, i, f, 4, 2, 8, dtype=dtype)
        with pytest.raises(ValueError, match=match):
            ks.moe.permute_backward(rows, pairs, i, 4, 2, 8, dtype=dtype)
        with pytest.raises(ValueError, match=match):
            ks.moe.gate_softmax_topk_backward(rows, f, f, i, rows, 4, 8, 2, dtype=dtype)
    with pytest.raises(ValueError, match="as dtype says"):     # beside raw addresses too
        ks.moe.permute_backward(4096, pairs, i, 4, 2, 8, dtype=ks.DType.F32)
