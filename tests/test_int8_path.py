"""CPU tests of the 8-bit activation path: what its entry points refuse, before anything reaches a GPU."""
import ctypes as C
import math

import pytest
import torch

from mixed_gemv_b200 import _lib, api
from mixed_gemv_b200.enums import DType, Status

A = 0x10000  # an address that no refused call may touch


def _norm(**kw):
    lib = _lib.load()
    a = _lib.RmsNormArgs()
    lib.mgv_rmsnorm_args_init(C.byref(a))
    for name in ("x", "weight", "q", "scale"):
        setattr(a, name, A)
    a.M, a.K, a.dtype = 4, 64, int(DType.F16)
    a.ldx = a.ldr = a.ldro = a.ldq = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.mgv_rmsnorm_quantize(C.byref(a), None)


def _gemm(**kw):
    lib = _lib.load()
    a = _lib.GemmI8Args()
    lib.mgv_gemm_i8_args_init(C.byref(a))
    for name in ("x", "weights", "x_scale", "weight_scale", "out"):
        setattr(a, name, A)
    a.M, a.N, a.K, a.ldx, a.ldw, a.ldd = 4, 32, 64, 64, 64, 32
    a.out_dtype, a.scale_dtype = int(DType.F16), int(DType.F32)
    for k, v in kw.items():
        setattr(a, k, v)
    plan = C.c_void_p(1)
    st = lib.mgv_gemm_i8(C.byref(a), None)
    assert lib.mgv_gemm_i8_plan_create(C.byref(a), C.byref(plan)) == st and not plan.value
    return st


def test_struct_layouts_match_the_header():
    lib = _lib.load()
    for struct, init in ((_lib.RmsNormArgs, lib.mgv_rmsnorm_args_init), (_lib.GemmI8Args, lib.mgv_gemm_i8_args_init)):
        a = struct()
        init(C.byref(a))
        assert a.struct_size == C.sizeof(struct)
    a = _lib.RmsNormArgs()
    lib.mgv_rmsnorm_args_init(C.byref(a))
    assert a.eps == pytest.approx(1e-5)


@pytest.mark.parametrize("kw, status", [
    (dict(struct_size=8), Status.INVALID_ARGUMENT),
    (dict(dtype=int(DType.F32)), Status.UNSUPPORTED),
    (dict(M=-1), Status.INVALID_ARGUMENT),
    (dict(M=1 << 31), Status.INVALID_ARGUMENT),
    (dict(K=0), Status.INVALID_ARGUMENT),
    (dict(K=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31), Status.INVALID_ARGUMENT),
    (dict(flags=_lib.FLAG_ACT_RELU), Status.INVALID_ARGUMENT),
    (dict(eps=-1e-6), Status.INVALID_ARGUMENT),
    (dict(eps=math.nan), Status.INVALID_ARGUMENT),
    (dict(eps=math.inf), Status.INVALID_ARGUMENT),
    (dict(x=None), Status.INVALID_ARGUMENT),
    (dict(weight=None), Status.INVALID_ARGUMENT),
    (dict(q=None), Status.INVALID_ARGUMENT),
    (dict(scale=None), Status.INVALID_ARGUMENT),
    (dict(ldx=63), Status.INVALID_ARGUMENT),
    (dict(ldq=63), Status.INVALID_ARGUMENT),
    (dict(residual=A), Status.INVALID_ARGUMENT),
    (dict(residual_out=A), Status.INVALID_ARGUMENT),
    (dict(residual=A, residual_out=A, ldr=64, ldro=72), Status.INVALID_ARGUMENT),
    (dict(residual=2 * A, residual_out=A, ldro=72), Status.INVALID_ARGUMENT),
    (dict(x=A + 1), Status.MISALIGNED),
    (dict(scale=A + 2), Status.MISALIGNED),
])
def test_norm_refusals(kw, status):
    assert _norm(**kw) == status
    assert b"rmsnorm_quantize" in _lib.load().mgv_last_error()


@pytest.mark.parametrize("kw, status", [
    (dict(struct_size=8), Status.INVALID_ARGUMENT),
    (dict(M=-1), Status.INVALID_ARGUMENT),
    (dict(M=(1 << 30) + 1), Status.INVALID_ARGUMENT),
    (dict(N=(1 << 30) + 1, ldd=1 << 31), Status.INVALID_ARGUMENT),
    (dict(N=0), Status.INVALID_ARGUMENT),
    (dict(K=0), Status.INVALID_ARGUMENT),
    (dict(K=131072, ldx=131072, ldw=131072), Status.INVALID_ARGUMENT),
    (dict(out_dtype=int(DType.F32)), Status.UNSUPPORTED),
    (dict(scale_dtype=3), Status.UNSUPPORTED),
    (dict(flags=_lib.FLAG_OUT_F32_PARTIAL), Status.INVALID_ARGUMENT),
    (dict(flags=_lib.FLAG_ACT_RELU | _lib.FLAG_ACT_SILU), Status.INVALID_ARGUMENT),
    (dict(flags=_lib.FLAG_ACT_RELU | _lib.FLAG_GATED_SILU), Status.INVALID_ARGUMENT),
    (dict(flags=_lib.FLAG_GATED_SILU, N=31), Status.INVALID_ARGUMENT),
    (dict(flags=_lib.FLAG_GATED_SILU, ldd=15), Status.INVALID_ARGUMENT),
    (dict(reserved=1), Status.INVALID_ARGUMENT),
    (dict(x=None), Status.INVALID_ARGUMENT),
    (dict(weights=None), Status.INVALID_ARGUMENT),
    (dict(x_scale=None), Status.INVALID_ARGUMENT),
    (dict(weight_scale=None), Status.INVALID_ARGUMENT),
    (dict(out=None), Status.INVALID_ARGUMENT),
    (dict(ldx=48), Status.INVALID_ARGUMENT),
    (dict(ldw=48), Status.INVALID_ARGUMENT),
    (dict(ldd=31), Status.INVALID_ARGUMENT),
    (dict(ldx=1 << 40), Status.INVALID_ARGUMENT),
    (dict(ldx=72), Status.MISALIGNED),
    (dict(ldw=72), Status.MISALIGNED),
    (dict(x=A + 8), Status.MISALIGNED),
    (dict(weights=A + 8), Status.MISALIGNED),
    (dict(x_scale=A + 2), Status.MISALIGNED),
    (dict(weight_scale=A + 2), Status.MISALIGNED),
    (dict(bias=A + 1), Status.MISALIGNED),
    (dict(out=A + 1), Status.MISALIGNED),
])
def test_gemm_refusals(kw, status):
    assert _gemm(**kw) == status
    assert b"gemm_i8" in _lib.load().mgv_last_error()


def test_row_call_refusals():
    lib = _lib.load()
    f16, f32 = int(DType.F16), int(DType.F32)
    for fn, name in ((lib.mgv_quantize_rows, b"quantize_rows"), (lib.mgv_dequantize_rows, b"dequantize_rows")):
        ok = [A, A, A, f16, 4, 64, 64, 64, 0, None]
        for at, value, status in ((0, None, Status.INVALID_ARGUMENT), (1, None, Status.INVALID_ARGUMENT),
                                  (2, None, Status.INVALID_ARGUMENT), (3, f32, Status.UNSUPPORTED),
                                  (4, -1, Status.INVALID_ARGUMENT), (5, 0, Status.INVALID_ARGUMENT),
                                  (6, 63, Status.INVALID_ARGUMENT), (7, 63, Status.INVALID_ARGUMENT),
                                  (8, _lib.FLAG_ACT_SILU, Status.INVALID_ARGUMENT)):
            args = list(ok)
            args[at] = value
            assert fn(*args) == status, (name, at)
            assert name in lib.mgv_last_error()
    assert lib.mgv_quantize_rows(A, A, A + 1, f16, 4, 64, 64, 64, 0, None) == Status.MISALIGNED
    assert lib.mgv_dequantize_rows(A, A, A + 1, f16, 4, 64, 64, 64, 0, None) == Status.MISALIGNED


def test_no_rows_need_no_gpu_and_no_buffers():
    lib = _lib.load()
    assert lib.mgv_quantize_rows(None, None, None, 0, 0, 64, 64, 64, 0, None) == Status.OK
    assert lib.mgv_dequantize_rows(None, None, None, 1, 0, 64, 64, 64, 0, None) == Status.OK
    assert _norm(M=0, x=None, weight=None, q=None, scale=None) == Status.OK


def test_plan_calls_take_null():
    lib = _lib.load()
    assert lib.mgv_gemm_i8_plan_create(None, None) == Status.INVALID_ARGUMENT
    assert lib.mgv_gemm_i8_plan_run(None, None) == Status.INVALID_ARGUMENT
    lib.mgv_gemm_i8_plan_destroy(None)


def test_python_face_refuses_host_tensors_and_unready_objects():
    h, q, s = torch.zeros(2, 16, dtype=torch.float16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    for op, args in ((api.RowQuantizer(), api.RowQuantizeArguments(x=h, q=q, scale=s)),
                     (api.RowDequantizer(), api.RowDequantizeArguments(q=q, scale=s, out=h)),
                     (api.RmsNormQuantizer(), api.RmsNormQuantizeArguments(x=h, weight=h[0], q=q, scale=s)),
                     (api.GemmI8Adaptor(), api.GemmI8Arguments(x=q, x_scale=s, weights=q, weight_scale=s, out=h[:, :2]))):
        with pytest.raises(api.MgvError, match="CUDA tensor"):
            op.initialize(args)
        with pytest.raises(api.MgvError, match="before initialize"):
            op.run()
