"""Host-only checks of the operators of language models: what their entry points
refuse, with which status, before any GPU work, and what the bindings check."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from ilgpu_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "operator_tests")
FAKE = 0x10000   # a non-null, aligned "device pointer" that is never dereferenced
BIG = 1 << 40
ONE = ctypes.byref(ctypes.c_float(1.0))


def number(x):
    return ctypes.byref(ctypes.c_float(x))


def test_bfloat16_is_a_type_of_its_own():
    assert capi.type_code(capi.bfloat16) == capi.BF16 == 11
    assert capi.type_code(np.uint16) == capi.U16 and capi.bfloat16.itemsize == 2
    # the primitives refuse it
    L = capi.lib()
    out = ctypes.c_int64()
    assert L.ilgpu_hip_radix_sort_temp_bytes(16, capi.BF16, 0, ctypes.byref(out)) == capi.ERROR_NOT_SUPPORTED
    assert L.ilgpu_hip_unique_temp_bytes(16, capi.BF16, ctypes.byref(out)) == capi.ERROR_NOT_SUPPORTED
    assert L.ilgpu_hip_transform(None, FAKE, 16, 1, capi.BF16, FAKE, 16, 1, capi.F32, 0, 0) == capi.ERROR_NOT_SUPPORTED
    assert L.ilgpu_hip_sequence(None, FAKE, 16, 1, capi.BF16, 1, 1) == capi.ERROR_NOT_SUPPORTED
    assert L.ilgpu_hip_histogram(None, FAKE, 16, 1, capi.BF16, FAKE, 16, capi.I32, 0, None) == capi.ERROR_NOT_SUPPORTED


def test_embedding_argument_validation():
    def call(table=FAKE, v=10, d=8, ts=8, tt=capi.F32, tokens=FAKE, n=4, kt=capi.I64, scale=ONE,
             out=FAKE, os_=8, ot=capi.BF16):
        return capi.lib().ilgpu_hip_embedding(None, table, v, d, ts, tt, tokens, n, kt, scale,
                                              out, os_, ot)

    assert call(tt=capi.F64) == call(ot=capi.F64) == call(tt=capi.I32) == call(ot=42) == capi.ERROR_NOT_SUPPORTED
    assert call(kt=capi.U32) == call(kt=capi.F32) == call(kt=capi.I16) == capi.ERROR_NOT_SUPPORTED
    assert call(table=None) == call(tokens=None) == call(out=None) == call(d=0) == capi.ERROR_NULL_VIEW
    assert call(n=-1) == call(v=-1) == call(d=-8) == call(ts=-1) == call(os_=7) == capi.ERROR_OUT_OF_RANGE
    assert call(n=1 << 31) == call(v=1 << 31) == call(d=1 << 31, os_=1 << 31) == capi.ERROR_NOT_SUPPORTED
    assert call(table=FAKE + 2) == call(tokens=FAKE + 4) == call(out=FAKE + 1) == capi.ERROR_NOT_SUPPORTED
    # nothing to do is no error, and needs no buffers
    assert call(n=0, tokens=None, out=None) == capi.SUCCESS
    assert call(n=0, tokens=None, out=None, table=None, v=0, scale=None) == capi.SUCCESS


def test_embedding_gradient_argument_validation():
    def call(go=FAKE, gs=8, gt=capi.BF16, tokens=FAKE, n=4, kt=capi.I32, scale=ONE, pad=-1, acc=0,
             table=FAKE, v=10, d=8, ts=8, tt=capi.F32, temp=FAKE, tb=BIG):
        return capi.lib().ilgpu_hip_embedding_gradient(
            None, go, gs, gt, tokens, n, kt, scale, pad, acc, table, v, d, ts, tt, temp, tb)

    assert call(gt=capi.F64) == call(tt=capi.F64) == call(kt=capi.U64) == capi.ERROR_NOT_SUPPORTED
    assert call(go=None) == call(tokens=None) == call(table=None) == call(d=0) == capi.ERROR_NULL_VIEW
    assert call(temp=None) == call(tb=0) == capi.ERROR_NULL_VIEW
    assert call(temp=FAKE + 2) == capi.ERROR_UNALIGNED_TEMP
    need = capi.embedding_gradient_temp_bytes(4, 10, 8)
    assert call(tb=need - 1) == call(gs=-1) == call(ts=7) == call(n=-1) == capi.ERROR_OUT_OF_RANGE
    assert call(n=1 << 31) == call(v=1 << 31) == call(table=FAKE + 2) == call(go=FAKE + 1) == capi.ERROR_NOT_SUPPORTED
    # no table rows, nothing to write
    assert call(v=0, table=None) == capi.SUCCESS
    for bad in ((-1, 1, 1), (1, -1, 1), (1, 1, 0)):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.embedding_gradient_temp_bytes(*bad)
    with pytest.raises(capi.NotSupportedError):
        capi.embedding_gradient_temp_bytes(1, 1 << 31, 1)


@pytest.mark.parametrize("vocabulary", [1, 1000, 50_000, 1 << 18, (1 << 18) + 1, 1 << 19, 1 << 20,
                                        (1 << 20) + 1, (1 << 31) - 1])
@pytest.mark.parametrize("dimension", [1, 64, 256, 257, 512, 769, 1024, 2048, 4096, 8192, 300_000])
def test_a_temp_of_the_embedding_gradient_serves_fewer_tokens(dimension, vocabulary):
    most = 0
    steps = [(1 << k) + more for k in range(18, 31) for more in (-1, 0, 1)]
    near = [(1 << k) + more for k in range(11, 18) for more in (-33, -32, -31, -1, 0, 1, 31, 32)]
    for n in sorted([*range(2100), *range(2100, 140_000, 31), *near, *steps]):
        need = capi.embedding_gradient_temp_bytes(n, vocabulary, dimension)
        assert need >= most, n
        most = need


def test_embedding_gradient_is_refused_where_sorts_are():
    L = capi.lib()
    capi.sort_set_parameter(capi.SORT_PARAM_ASSUME_LDS_ATOMIC_ORDER, 0)
    try:
        for n, v in ((4, 10), (1 << 20, 10), (100, 1 << 30)):
            assert L.ilgpu_hip_embedding_gradient(
                None, FAKE, 8, capi.F32, FAKE, n, capi.I32, ONE, -1, 0, FAKE, v, 8, 8, capi.F32,
                FAKE, BIG) == capi.ERROR_NOT_SUPPORTED
    finally:
        capi.sort_set_parameter(capi.SORT_PARAM_ASSUME_LDS_ATOMIC_ORDER, -1)


def test_embedding_gradient_of_more_sums_than_a_grid_holds():
    # Broadcast rows take no memory, but 2^31 - 1 positions of 512 columns want 2^25 blocks of 256.
    L, n = capi.lib(), (1 << 31) - 1
    assert capi.embedding_gradient_temp_bytes(n, 10, 512) < BIG
    assert L.ilgpu_hip_embedding_gradient(
        None, FAKE, 0, capi.F32, FAKE, n, capi.I32, ONE, -1, 0, FAKE, 10, 512, 512, capi.F32,
        FAKE, BIG) == capi.ERROR_NOT_SUPPORTED


def test_layer_norm_argument_validation():
    def call(x=FAKE, r=4, c=8, xs=8, t=capi.F16, w=FAKE, b=FAKE, wt=capi.F32, eps=number(1e-5),
             out=FAKE, os_=8, mean=FAKE, rstd=FAKE):
        return capi.lib().ilgpu_hip_layer_norm(None, x, r, c, xs, t, w, b, wt, eps, out, os_, mean,
                                               rstd)

    assert call(t=capi.F64, wt=capi.F64) == call(wt=capi.BF16) == call(t=capi.F32, wt=capi.F16) == capi.ERROR_NOT_SUPPORTED
    assert call(t=capi.I32) == capi.ERROR_NOT_SUPPORTED
    assert call(x=None) == call(out=None) == call(c=0) == call(eps=None) == capi.ERROR_NULL_VIEW
    assert call(r=-1) == call(c=-1) == call(xs=-1) == call(os_=7) == capi.ERROR_OUT_OF_RANGE
    for bad in (-1e-5, float("nan"), float("inf")):
        assert call(eps=number(bad)) == capi.ERROR_OUT_OF_RANGE
    assert call(r=1 << 31) == call(x=FAKE + 1) == call(w=FAKE + 2) == call(b=FAKE + 1) == capi.ERROR_NOT_SUPPORTED
    assert call(mean=FAKE + 2) == call(rstd=FAKE + 2) == capi.ERROR_NOT_SUPPORTED
    assert call(r=0, x=None, out=None, w=None, b=None, mean=None, rstd=None) == capi.SUCCESS


def test_layer_norm_gradient_argument_validation():
    def call(go=FAKE, gs=8, x=FAKE, xs=8, r=4, c=8, t=capi.BF16, w=FAKE, wt=capi.BF16, mean=FAKE,
             rstd=FAKE, gi=FAKE, gis=8, gw=FAKE, gb=FAKE, acc=0, temp=FAKE, tb=BIG):
        return capi.lib().ilgpu_hip_layer_norm_gradient(
            None, go, gs, x, xs, r, c, t, w, wt, mean, rstd, gi, gis, gw, gb, acc, temp, tb)

    assert call(t=capi.F64) == call(wt=capi.F16) == call(t=capi.U8) == capi.ERROR_NOT_SUPPORTED
    assert call(go=None) == call(x=None) == call(mean=None) == call(rstd=None) == call(c=0) == capi.ERROR_NULL_VIEW
    assert call(gi=None, gw=None, gb=None) == call(temp=None) == call(tb=-4) == capi.ERROR_NULL_VIEW
    assert call(gis=7) == call(gs=-1) == call(xs=-1) == call(r=-1) == capi.ERROR_OUT_OF_RANGE
    assert call(tb=capi.layer_norm_gradient_temp_bytes(4, 8) - 1) == capi.ERROR_OUT_OF_RANGE
    assert call(temp=FAKE + 1) == capi.ERROR_UNALIGNED_TEMP
    assert call(c=1 << 31, gs=1 << 31) == call(gw=FAKE + 1) == call(gb=FAKE + 1) == call(mean=FAKE + 1) == capi.ERROR_NOT_SUPPORTED
    assert call(r=0, go=None, x=None, mean=None, rstd=None, gi=None, gw=None, gb=None) == capi.SUCCESS
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.layer_norm_gradient_temp_bytes(4, 0)
    with pytest.raises(capi.NotSupportedError):
        capi.layer_norm_gradient_temp_bytes(1 << 31, 4)


def table_of(*entries):
    return (capi._Tensor * max(1, len(entries)))(*entries)


def test_gradient_norm_and_clip_argument_validation():
    L = capi.lib()
    good = table_of((FAKE, 10, capi.F32, 0), (None, 0, capi.F16, 0), (FAKE, 3, capi.BF16, 0))

    def norm(tensors=good, n=3, out=FAKE, temp=FAKE, tb=BIG):
        return L.ilgpu_hip_gradient_norm(None, tensors, n, out, temp, tb)

    def clip(tensors=good, targets=None, n=3, norm_=FAKE, limit=number(1.0)):
        return L.ilgpu_hip_clip_gradients(None, tensors, targets, n, norm_, limit)

    assert norm(out=None) == norm(temp=None) == norm(tensors=None) == capi.ERROR_NULL_VIEW
    assert norm(n=-1) == norm(tb=capi.gradient_norm_temp_bytes(3) - 1) == capi.ERROR_OUT_OF_RANGE
    assert norm(temp=FAKE + 2) == capi.ERROR_UNALIGNED_TEMP
    assert norm(out=FAKE + 2) == capi.ERROR_NOT_SUPPORTED
    assert clip(tensors=None) == clip(norm_=None) == clip(limit=None) == capi.ERROR_NULL_VIEW
    assert clip(limit=number(-1.0)) == clip(limit=number(float("nan"))) == clip(n=-2) == capi.ERROR_OUT_OF_RANGE
    assert clip(norm_=FAKE + 1) == capi.ERROR_NOT_SUPPORTED
    for entry, status in (((FAKE, 10, capi.F64, 0), capi.ERROR_NOT_SUPPORTED),
                          ((FAKE, 10, capi.I32, 0), capi.ERROR_NOT_SUPPORTED),
                          ((FAKE, -1, capi.F32, 0), capi.ERROR_OUT_OF_RANGE),
                          ((None, 10, capi.F32, 0), capi.ERROR_NULL_VIEW),
                          ((FAKE + 2, 10, capi.F32, 0), capi.ERROR_NOT_SUPPORTED),
                          ((FAKE, (1 << 40) + 1, capi.F32, 0), capi.ERROR_NOT_SUPPORTED)):
        bad = table_of((FAKE, 5, capi.F32, 0), entry)
        assert norm(tensors=bad, n=2) == clip(tensors=bad, n=2) == status
        assert clip(tensors=table_of((FAKE, 5, capi.F32, 0), (FAKE, 10, capi.F32, 0)),
                    targets=bad, n=2) == status
    # targets of another length or type
    assert clip(targets=table_of((FAKE, 9, capi.F32, 0), (None, 0, capi.F16, 0), (FAKE, 3, capi.BF16, 0))) == capi.ERROR_OUT_OF_RANGE
    assert clip(targets=table_of((FAKE, 10, capi.F32, 0), (None, 0, capi.F16, 0), (FAKE, 3, capi.F16, 0))) == capi.ERROR_NOT_SUPPORTED
    # a list of nothing scales nothing
    assert clip(tensors=None, n=0) == clip(tensors=table_of((None, 0, capi.F32, 0)), n=1) == capi.SUCCESS
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.gradient_norm_temp_bytes(-1)


def host_array(length, dtype):
    """A DeviceArray on host memory, for checks that come before any call."""
    import torch
    return capi.DeviceArray(length, dtype, _bytes=torch.zeros(
        max(1, length * np.dtype(dtype).itemsize), dtype=torch.uint8))


def test_the_bindings_checks_of_views():
    f32, bf16 = np.float32, capi.bfloat16
    M, A = capi.DeviceMatrix, host_array
    with pytest.raises(capi.ArgumentOutOfRangeError):
        M(A(15, f32), 4, 4)
    with pytest.raises(capi.ArgumentOutOfRangeError):
        M(A(16, f32), 4, 4, 5)
    with pytest.raises(capi.ArgumentOutOfRangeError):
        M(A(16, f32), 4, 4, -4)
    assert M(A(19, f32), 4, 4, 5).row_stride == 5 and M(A(4, f32), 9, 4, 0).rows == 9
    table, tokens = M(A(40, f32), 10, 4), A(3, np.int64)
    for out in (M(A(8, f32), 2, 4), M(A(9, f32), 3, 3)):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.embedding(table, tokens, out, stream=0)
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.embedding_gradient(out, tokens, table, A(100, np.int32), stream=0)
    with pytest.raises(capi.NotSupportedError):
        capi.embedding(table, A(6, np.int64).strided(2), M(A(12, f32), 3, 4), stream=0)
    x, y = M(A(12, f32), 3, 4), M(A(12, f32), 3, 4)
    for kw in ({"weight": A(5, f32)}, {"bias": A(3, f32)}, {"mean": A(2, f32)}, {"rstd": A(2, f32)}):
        with pytest.raises(capi.ArgumentOutOfRangeError):
            capi.layer_norm(x, y, stream=0, **kw)
    for kw in ({"weight": A(4, f32), "bias": A(4, np.float16)}, {"mean": A(3, np.float64)}):
        with pytest.raises(capi.NotSupportedError):
            capi.layer_norm(x, y, stream=0, **kw)
    with pytest.raises(capi.NotSupportedError):
        capi.layer_norm(x, M(A(12, bf16), 3, 4), stream=0)
    stat = A(3, f32)
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.layer_norm_gradient(M(A(8, f32), 2, 4), x, None, stat, stat, y, stream=0)
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.layer_norm_gradient(y, x, None, stat, stat, None, A(5, f32), None, A(99, np.int32), stream=0)
    with pytest.raises(capi.NotSupportedError):
        capi.layer_norm_gradient(y, x, None, stat, stat, M(A(12, bf16), 3, 4), stream=0)
    with pytest.raises(capi.NotSupportedError):
        capi.gradient_norm([A(4, f32).strided(2)], A(1, f32), A(99, np.int32), stream=0)
    with pytest.raises(capi.NotSupportedError):
        capi.clip_gradients([A(4, f32)], A(1, np.float64), 1.0, stream=0)
    with pytest.raises(capi.ArgumentOutOfRangeError):
        capi.clip_gradients([A(4, f32)], A(1, f32), 1.0, [], stream=0)


def test_a_matrix_is_made_of_a_dense_array():
    # the elements of a strided view do not lie side by side, as those of a row do
    M, A = capi.DeviceMatrix, host_array
    for rows, columns, stride in ((2, 4, 4), (1, 8, None), (8, 1, 1), (5, 8, 0)):
        with pytest.raises(capi.NotSupportedError):
            M(A(32, np.float32).strided(2), rows, columns, stride)
    assert M(A(32, np.float32).strided(1), 8, 4).rows == 8


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
