"""Host-only checks of the gated recurrence, the residual norm and the AdamW step: what
their entry points refuse, with which status, before any GPU work, and what the bindings
check."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from ilgpu_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "recurrent_operator_tests")
FAKE = 0x10000   # a non-null, aligned "device pointer" that is never dereferenced
BIG = 1 << 40
NULL, RANGE, UNSUPPORTED = capi.ERROR_NULL_VIEW, capi.ERROR_OUT_OF_RANGE, capi.ERROR_NOT_SUPPORTED


def number(x):
    return ctypes.byref(ctypes.c_float(x))


def all_are(status, *got):
    assert got == (status,) * len(got)


def test_recurrence_argument_validation():
    def call(gate=FAKE, gs=8, x=FAKE, xs=8, r=600, c=8, t=capi.BF16, decay=0, complement=1,
             offsets=FAKE, ot=capi.I32, n=3, first=FAKE, fs=8, out=FAKE, os_=8, last=FAKE, ls=8,
             temp=FAKE, tb=BIG):
        return capi.lib().ilgpu_hip_gated_recurrence(
            None, gate, gs, x, xs, r, c, t, decay, complement, offsets, ot, n, first, fs, out, os_, last, ls,
            temp, tb)

    all_are(UNSUPPORTED, call(t=capi.F64), call(t=capi.I32), call(t=42), call(decay=2), call(decay=-1),
            call(ot=capi.U32), call(ot=capi.F32), call(r=1 << 31), call(n=(1 << 31) - 1),
            call(gate=FAKE + 1), call(x=FAKE + 1), call(out=FAKE + 1), call(first=FAKE + 2),
            call(last=FAKE + 2), call(offsets=FAKE + 2), call(offsets=FAKE + 4, ot=capi.I64))
    all_are(NULL, call(gate=None), call(x=None), call(out=None), call(c=0), call(temp=None), call(tb=0))
    all_are(RANGE, call(r=-1), call(c=-1), call(n=-1), call(gs=-1), call(xs=-1), call(os_=7), call(fs=-1),
            call(ls=7), call(tb=capi.gated_recurrence_temp_bytes(600, 8) - 1),
            call(offsets=None, n=7), call(offsets=None, n=0), call(offsets=None, n=601))
    assert call(temp=FAKE + 2) == capi.ERROR_UNALIGNED_TEMP
    # nothing to do is no error, and needs no buffers
    all_are(capi.SUCCESS, call(r=0, gate=None, x=None, out=None, last=None, temp=None, tb=0),
            call(r=0, n=0, gate=None, x=None, out=None, first=None, last=None, offsets=None, temp=None, tb=0))
    for bad in ((-1, 1), (1, 0), (1, -1)):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.gated_recurrence_temp_bytes(*bad)
    with pytest.raises(capi.NotSupportedError):
        capi.gated_recurrence_temp_bytes(1 << 31, 1)


def test_recurrence_gradient_argument_validation():
    def call(go=FAKE, gos=8, gate=FAKE, gs=8, x=FAKE, xs=8, out=FAKE, os_=8, r=600, c=8, t=capi.F16, decay=1,
             complement=0, offsets=None, ot=capi.I32, n=3, first=FAKE, fs=8, gf=FAKE, gfs=8, gg=FAKE, ggs=8,
             gx=FAKE, gxs=8, gi=FAKE, gis=8, temp=FAKE, tb=BIG):
        return capi.lib().ilgpu_hip_gated_recurrence_gradient(
            None, go, gos, gate, gs, x, xs, out, os_, r, c, t, decay, complement, offsets, ot, n, first, fs, gf,
            gfs, gg, ggs, gx, gxs, gi, gis, temp, tb)

    all_are(UNSUPPORTED, call(t=capi.F64), call(decay=7), call(go=FAKE + 1), call(gg=FAKE + 1), call(gx=FAKE + 1),
            call(gi=FAKE + 2), call(gf=FAKE + 1), call(out=FAKE + 1))
    all_are(NULL, call(go=None), call(gate=None), call(x=None), call(out=None), call(gg=None, gx=None, gi=None),
            call(temp=None))
    all_are(RANGE, call(gos=-1), call(os_=-1), call(ggs=7), call(gxs=7), call(gis=7), call(gfs=-1), call(n=7),
            call(tb=4))
    # (one row in the place of all is fine where it is read)
    assert call(r=0, n=0, go=None, gate=None, x=None, out=None, gg=None, gx=None, gi=None, first=None, gf=None,
                temp=None) == capi.SUCCESS


@pytest.mark.parametrize("channels", [1, 7, 8, 64, 65, 4096])
def test_a_temp_of_the_recurrence_serves_fewer_rows(channels):
    most = 0
    for n in [*range(3000), *((1 << k) + more for k in range(12, 31) for more in (-1, 0, 1))]:
        need = capi.gated_recurrence_temp_bytes(n, channels)
        assert need >= most, n
        most = need


@pytest.mark.parametrize("columns", [1, 64, 4096, 4097, 8192, 100_000])
def test_a_temp_of_the_norms_gradient_serves_fewer_rows(columns):
    most = 0
    for n in [*range(3000), *((1 << k) + more for k in range(12, 31) for more in (-1, 0, 1))]:
        need = capi.residual_norm_gradient_temp_bytes(n, columns)
        assert need >= most, n
        most = need


def test_residual_norm_argument_validation():
    def call(x=FAKE, xs=8, r=4, c=8, t=capi.BF16, norm=1, iw=FAKE, gate=FAKE, gs=8, gk=1, res=FAKE, rs=8,
             rt=capi.F32, scale=number(0.5), w=FAKE, wt=capi.F32, eps=number(1e-5), total=FAKE, ts=8, out=FAKE,
             os_=8, irstd=FAKE, rstd=FAKE):
        return capi.lib().ilgpu_hip_residual_norm(
            None, x, xs, r, c, t, norm, iw, gate, gs, gk, res, rs, rt, scale, w, wt, eps, total, ts, out, os_,
            irstd, rstd)

    all_are(UNSUPPORTED, call(t=capi.F64), call(rt=capi.F16), call(wt=capi.F16), call(t=capi.F32, rt=capi.BF16),
            call(gk=2), call(gk=-1), call(x=FAKE + 1), call(gate=FAKE + 1), call(res=FAKE + 2), call(total=FAKE + 2),
            call(out=FAKE + 1), call(w=FAKE + 2), call(iw=FAKE + 2), call(irstd=FAKE + 2), call(rstd=FAKE + 1),
            call(r=1 << 31))
    all_are(NULL, call(x=None), call(c=0), call(eps=None), call(total=None, out=None))
    all_are(RANGE, call(r=-1), call(xs=-1), call(gs=-1), call(rs=-1), call(ts=7), call(os_=7),
            call(eps=number(-1.0)), call(eps=number(float("nan"))), call(eps=number(float("inf"))))
    assert call(r=0, x=None, gate=None, res=None, total=None, out=None, w=None, iw=None, scale=None,
                irstd=None, rstd=None) == capi.SUCCESS


def test_residual_norm_gradient_argument_validation():
    def call(go=FAKE, gos=8, gt=FAKE, gts=8, x=FAKE, xs=8, r=4, c=8, t=capi.F16, norm=1, iw=FAKE, irstd=FAKE,
             gate=FAKE, gs=8, gk=0, total=FAKE, ts=8, rt=capi.F16, scale=None, w=FAKE, wt=capi.F16, rstd=FAKE,
             gx=FAKE, gxs=8, gg=FAKE, ggs=8, gr=FAKE, grs=8, giw=FAKE, gw=FAKE, acc=0, temp=FAKE, tb=BIG):
        return capi.lib().ilgpu_hip_residual_norm_gradient(
            None, go, gos, gt, gts, x, xs, r, c, t, norm, iw, irstd, gate, gs, gk, total, ts, rt, scale, w, wt, rstd,
            gx, gxs, gg, ggs, gr, grs, giw, gw, acc, temp, tb)

    all_are(UNSUPPORTED, call(t=capi.F64), call(rt=capi.BF16), call(wt=capi.BF16), call(gk=3), call(go=FAKE + 1),
            call(gt=FAKE + 1), call(gx=FAKE + 1), call(gg=FAKE + 1), call(gr=FAKE + 1), call(gw=FAKE + 1),
            call(giw=FAKE + 1), call(total=FAKE + 1), call(rstd=FAKE + 2), call(irstd=FAKE + 2))
    all_are(NULL, call(x=None), call(c=0), call(go=None, gt=None), call(total=None), call(rstd=None),
            call(irstd=None), call(gate=None), call(go=None), call(norm=0),
            call(gx=None, gg=None, gr=None, giw=None, gw=None), call(temp=None))
    all_are(RANGE, call(gos=-1), call(gts=-1), call(xs=-1), call(ts=-1), call(gs=-1), call(gxs=7), call(ggs=7),
            call(grs=7), call(r=-1), call(tb=capi.residual_norm_gradient_temp_bytes(4, 8) - 1))
    assert call(temp=FAKE + 2) == capi.ERROR_UNALIGNED_TEMP
    for bad in ((-1, 1), (1, 0)):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.residual_norm_gradient_temp_bytes(*bad)


def table_of(*entries):
    return (capi._Tensor * max(1, len(entries)))(*entries)


def options(**more):
    o = dict(rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.1, max_norm=1.0, seed=0, **{})
    o.update(more)
    return ctypes.byref(capi._AdamwOptions(**o))


def test_adamw_argument_validation():
    def floats(kind=capi.F32, a=FAKE, n=300):
        return table_of((a, n, kind, 0), (None, 0, kind, 0))

    def call(p=floats(), g=floats(capi.BF16), m=floats(), v=floats(), ms=None, vs=None, c=None, n=2, o=options(),
             step=FAKE, schedule=FAKE, norm=FAKE):
        return capi.lib().ilgpu_hip_adamw(None, p, g, m, v, ms, vs, c, n, o, step, schedule, norm)

    codes, scales = floats(capi.U8, FAKE + 1), floats(n=2)
    all_are(NULL, call(p=None), call(g=None), call(m=None), call(v=None), call(o=None), call(step=None),
            call(ms=scales), call(vs=scales), call(p=floats(a=None)), call(g=floats(a=None)),
            call(c=floats(a=None)), call(m=codes, v=codes, ms=floats(a=None, n=2), vs=scales))
    all_are(UNSUPPORTED, call(p=floats(capi.F64)), call(g=floats(capi.I32)), call(m=floats(capi.BF16)),
            call(v=floats(capi.U8)), call(c=floats(capi.U8)), call(p=floats(a=FAKE + 2)), call(g=floats(capi.F16, FAKE + 1)),
            call(m=floats(a=FAKE + 1)), call(step=FAKE + 4), call(schedule=FAKE + 2), call(norm=FAKE + 1),
            call(ms=scales, vs=scales), call(m=codes, v=codes, ms=floats(capi.F16, n=2), vs=scales),
            call(p=floats(n=(1 << 40) + 1)))
    all_are(RANGE, call(n=-1), call(g=floats(n=299)), call(m=floats(n=301)), call(v=floats(n=2)), call(c=floats(n=1)),
            call(m=codes, v=codes, ms=floats(n=1), vs=scales), call(m=codes, v=codes, ms=scales, vs=floats(n=3)),
            *(call(o=options(**{k: bad})) for k in ("rate", "beta1", "beta2", "epsilon", "weight_decay", "max_norm")
              for bad in (-0.5, float("nan"))),
            *(call(o=options(**{k: 1.0})) for k in ("beta1", "beta2")), call(o=options(beta2=1 - 1e-12)),
            *(call(o=options(**{k: float("inf")})) for k in ("rate", "epsilon", "weight_decay")),
            call(o=options(epsilon=0.0)), call(o=options(epsilon=1e-39)))
    # a list of nothing steps nothing
    none = table_of((None, 0, capi.F32, 0))
    all_are(capi.SUCCESS, call(p=none, g=none, m=none, v=none, n=1), call(n=0, p=None, g=None, m=None, v=None))


def test_adamw_moments_argument_validation():
    def one(kind, n, a=FAKE):
        return table_of((a, n, kind, 0))

    def call(m=one(capi.U8, 300), ms=one(capi.F32, 2), mt=one(capi.BF16, 300), v=None, vs=None, vt=None, n=1):
        return capi.lib().ilgpu_hip_adamw_moments(None, m, ms, mt, v, vs, vt, n)

    all_are(NULL, call(m=None), call(ms=None), call(mt=None), call(m=None, ms=None, mt=None), call(v=one(capi.U8, 300)))
    all_are(UNSUPPORTED, call(m=one(capi.F32, 300)), call(ms=one(capi.F16, 2)), call(mt=one(capi.U8, 300)),
            call(mt=one(capi.F32, 300, FAKE + 2)))
    all_are(RANGE, call(m=one(capi.U8, 299)), call(ms=one(capi.F32, 1)), call(n=-1))
    assert call(m=None, ms=None, mt=None, n=0) == capi.SUCCESS


def host_array(length, dtype):
    """A DeviceArray on host memory, for checks that come before any call."""
    import torch
    return capi.DeviceArray(length, dtype, _bytes=torch.zeros(
        max(1, length * np.dtype(dtype).itemsize), dtype=torch.uint8))


def test_the_bindings_checks():
    f32, bf16 = np.float32, capi.bfloat16
    A = host_array

    def M(rows, columns, kind=f32):
        return capi.DeviceMatrix(A(rows * columns, kind), rows, columns)

    x = M(6, 4)
    for bad in (dict(gate=M(5, 4)), dict(out=M(6, 3)), dict(initial=M(3, 4)), dict(final=M(2, 5)),
                dict(offsets=A(2, np.int32))):
        args = dict(gate=x, inp=x, out=x, sequences=2, stream=0, temp=A(9, np.int32))
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.gated_recurrence(**{**args, **bad})
    for bad in (dict(gate=M(6, 4, bf16)), dict(initial=M(2, 4, np.float64)),
                dict(offsets=A(6, np.int32).strided(2))):
        with pytest.raises(capi.NotSupportedError):
            capi.gated_recurrence(**{**args, **bad})
    args = dict(grad_out=x, gate=x, inp=x, out=x, grad_gate=x, grad_in=None, sequences=2, stream=0)
    for bad in (dict(grad_gate=M(6, 5)), dict(grad_in=M(1, 4)), dict(grad_final=M(1, 4)), dict(grad_initial=M(2, 3))):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.gated_recurrence_gradient(**{**args, **bad})
    args = dict(inp=x, residual=x, total=x, out=x, stream=0)
    for bad in (dict(residual=M(5, 4)), dict(total=M(6, 5)), dict(out=M(7, 4)), dict(gate=M(6, 3)),
                dict(weight=A(3, f32)), dict(input_weight=A(5, f32)), dict(rstd=A(5, f32)), dict(input_rstd=A(5, f32))):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.residual_norm(**{**args, **bad})
    for bad in (dict(total=M(6, 4, bf16)), dict(gate=M(6, 4, bf16)), dict(out=M(6, 4, bf16)), dict(rstd=A(6, np.float64)),
                dict(weight=A(4, f32), input_weight=A(4, bf16))):
        with pytest.raises(capi.NotSupportedError):
            capi.residual_norm(**{**args, **bad})
    args = dict(grad_out=x, grad_total=x, inp=x, total=x, weight=None, rstd=A(6, f32), grad_in=x, stream=0,
                temp=A(9, np.int32))
    for bad in (dict(grad_out=M(5, 4)), dict(grad_total=M(6, 3)), dict(grad_residual=M(6, 3)), dict(grad_gate=M(1, 4)),
                dict(grad_weight=A(5, f32)), dict(rstd=A(5, f32))):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.residual_norm_gradient(**{**args, **bad})
    with pytest.raises(capi.NotSupportedError):
        capi.residual_norm_gradient(**{**args, "grad_residual": M(6, 4, bf16)})
    p, step = [A(4, f32)], A(1, np.int64)
    for bad in (dict(gradients=[]), dict(first=p + p), dict(second=[]), dict(copies=[]), dict(first_scales=[])):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.adamw(**{**dict(parameters=p, gradients=p, first=p, second=p, step=step, rate=0.1, stream=0), **bad})
    for bad in (dict(step=A(1, np.int32)), dict(norm=A(1, np.float64)), dict(gradients=[A(8, f32).strided(2)])):
        with pytest.raises(capi.NotSupportedError):
            capi.adamw(**{**dict(parameters=p, gradients=p, first=p, second=p, step=step, rate=0.1, stream=0), **bad})
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.adamw_moments([A(4, np.uint8)], [A(1, f32)], [], stream=0)


def run(*args):
    assert os.path.exists(BINARY), "build it with `python -m ilgpu_amd.build`"
    proc = subprocess.run([BINARY, *args], capture_output=True, text=True, timeout=300)
    print(proc.stdout[-4000:])
    print(proc.stderr[-2000:])
    return proc


def test_cpp_host_layer_checks():
    proc = run("--host")
    assert proc.returncode == 0 and "0 failed checks" in proc.stdout


@pytest.mark.gpu
def test_cpp_host_layer():
    proc = run()
    assert proc.returncode == 0 and "0 failed checks" in proc.stdout, proc.stdout[-2000:]
