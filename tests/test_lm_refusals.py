"""Calls of the operators around a language model that the library refuses before any CUDA call."""
import ctypes as C

import pytest

from bsipytorch_b200 import capi


class Plan(C.Structure):
    _fields_ = [("per", C.c_int64), ("block_stride", C.c_int64), ("row_stride", C.c_int64)]


PLAN = C.byref(Plan(0, 0, 64))
P = C.c_void_p(256)           # an address that nobody reads


def refused(rc, code=capi.ERR_INVALID):
    assert rc == code and capi.lib().bsi_b200_last_error()


def test_token_logprobs():
    f = capi.lib().bsi_b200_token_logprobs
    out = (P, P, P, P, P)
    refused(f(None, 0, 4, 64, PLAN, P, PLAN, 2, *out, None))              # null logits
    refused(f(P, 9, 4, 64, PLAN, P, PLAN, 2, *out, None))                 # dtype
    refused(f(P, 0, 4, 0, PLAN, P, PLAN, 0, *out, None))                  # no vocabulary
    refused(f(P, 0, -1, 64, PLAN, P, PLAN, 0, *out, None))
    refused(f(P, 0, 1 << 31, 64, PLAN, P, PLAN, 0, *out, None))
    refused(f(P, 0, 4, 64, None, P, PLAN, 0, *out, None))                 # no plan
    refused(f(P, 0, 4, 64, PLAN, P, None, 0, *out, None))
    refused(f(P, 0, 4, 64, PLAN, P, C.byref(Plan(-1, 0, 1)), 0, *out, None))
    refused(f(P, 0, 4, 64, C.byref(Plan(-(1 << 32), 0, 64)), P, PLAN, 0, *out, None))
    refused(f(P, 0, 4, 64, PLAN, P, PLAN, 65, *out, None))                # more alternatives than logits
    refused(f(P, 0, 4, 640, PLAN, P, PLAN, 129, *out, None))
    refused(f(P, 0, 4, 64, PLAN, P, PLAN, 2, P, P, P, None, P, None))     # nowhere to put them
    refused(f(C.c_void_p(257), 1, 4, 64, PLAN, P, PLAN, 2, *out, None))   # misaligned
    assert f(None, 0, 0, 64, PLAN, None, None, 2, None, None, None, None, None, None) == capi.OK


@pytest.mark.parametrize("name", ["forward", "fused"])
def test_distillation(name):
    f = getattr(capi.lib(), "bsi_b200_distill_" + name)

    def call(logits=P, dtype=0, rows=4, V=64, plan=PLAN, ids=P, teacher=P, teacher_dtype=0, K=5, T=1.0, row_loss=P, saved=P, loss=P, total=P, grad=P, stride=64):
        head = (logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, T, 0, None, 1, row_loss)
        return f(*head, saved, loss, total, None) if name == "forward" else f(*head, loss, total, grad, stride, None)

    for bad in (dict(logits=None), dict(dtype=3), dict(V=0), dict(plan=None), dict(ids=None), dict(teacher=None), dict(teacher_dtype=-1), dict(K=0), dict(K=513),
                dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(row_loss=None), dict(ids=C.c_void_p(260)),
                dict(teacher=C.c_void_p(258))):
        refused(call(**bad))
    for bad in (dict(saved=C.c_void_p(260)),) if name == "forward" else (dict(grad=None), dict(stride=63), dict(total=None), dict(loss=None)):
        refused(call(**bad))


def test_distillation_backward():
    f = capi.lib().bsi_b200_distill_backward

    def call(rows=4, saved=P, grad=P, stride=64, K=5):
        return f(P, 0, rows, 64, PLAN, P, P, 0, K, 1.0, 0, None, saved, None, 0, None, grad, stride, None)

    for bad in (dict(saved=None), dict(saved=C.c_void_p(264)), dict(grad=None), dict(stride=10), dict(K=0)):
        refused(call(**bad))
    assert call(rows=0, saved=None, grad=None) == capi.OK


def test_four_bit_matrices():
    L = capi.lib()
    assert L.bsi_b200_fp4_scale_bytes(1, 1, 0) == 1024 and L.bsi_b200_fp4_scale_bytes(129, 257, 1) == 2 * 8 * 512
    assert L.bsi_b200_fp4_scale_bytes(4, 0, 0) == -1 and L.bsi_b200_fp4_scale_bytes(4, 4, 2) == -1 and L.bsi_b200_fp4_scale_bytes(-1, 4, 1) == -1

    def pack(x=P, dtype=0, rows=4, K=64, format=1, codes=P, ld=32, scales=P, row=P):
        return L.bsi_b200_fp4_quantize(x, dtype, rows, K, K, format, codes, ld, scales, row, None)

    for bad in (dict(x=None), dict(dtype=3), dict(rows=-1), dict(K=0), dict(format=2), dict(codes=None), dict(ld=31), dict(ld=16), dict(scales=None), dict(row=None),
                dict(codes=C.c_void_p(264)), dict(x=C.c_void_p(257))):
        refused(pack(**bad))
    assert pack(x=None, rows=0, codes=None, scales=None, row=None) == capi.OK

    def unpack(out=P, ldo=64, dtype=0):
        return L.bsi_b200_fp4_dequantize(P, 32, P, P, 4, 64, 1, out, dtype, ldo, None)

    for bad in (dict(out=None), dict(ldo=63), dict(dtype=5), dict(out=C.c_void_p(257))):
        refused(unpack(**bad))

    def linear(M=4, N=8, K=64, xc=P, xs=P, xg=P, wc=P, ws=P, wg=P, ldx=32, ldw=32, format=1, y=P, ldy=8, dtype=0, act=0):
        return L.bsi_b200_fp4_linear(xc, ldx, xs, xg, wc, ldw, ws, wg, None, M, N, K, format, y, ldy, dtype, act, 0, None)

    for bad in (dict(M=-1), dict(N=-1), dict(K=0), dict(xc=None), dict(xs=None), dict(wc=None), dict(ws=None), dict(xg=None), dict(wg=None), dict(ldx=16), dict(ldw=40),
                dict(format=-1), dict(y=None), dict(ldy=7), dict(dtype=4), dict(act=2), dict(y=C.c_void_p(258)), dict(wc=C.c_void_p(264)), dict(M=1 << 24)):
        refused(linear(**bad))
    assert linear(M=0, y=None) == capi.OK and linear(N=0, ldy=0) == capi.OK


def test_names_are_checked_in_python():
    torch = pytest.importorskip("torch")
    from bsipytorch_b200 import microscale, scoring
    with pytest.raises(ValueError):
        microscale.quantize_fp4(torch.zeros(2, 2), "int4")
    with pytest.raises(ValueError):
        scoring.distillation_loss(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1), reduction="batchmean")
    with pytest.raises(RuntimeError):
        scoring.token_logprobs(torch.zeros(2, 4))
    with pytest.raises(RuntimeError):
        microscale.quantize_fp4(torch.zeros(2, 4))


@pytest.mark.parametrize("fmt,block", [("mxfp4", 32), ("nvfp4", 16)])
@pytest.mark.parametrize("rows,features", [(0, 96), (0, 1), (1, 1), (130, 300)])
def test_block_scales_of_any_number_of_rows(fmt, block, rows, features):
    torch = pytest.importorskip("torch")
    from bsipytorch_b200 import microscale
    n = capi.lib().bsi_b200_fp4_scale_bytes(rows, features, microscale.FORMATS[fmt])
    one = torch.full((n,), 127 if fmt == "mxfp4" else 0x38, dtype=torch.uint8)          # 1.0
    codes = torch.zeros(rows, -(-features // 32) * 16, dtype=torch.uint8)
    q = microscale.FP4Matrix(codes, one, None, features, fmt, torch.float32)
    assert torch.equal(q.block_scales(), torch.ones(rows, -(-features // block))) and q.shape == (rows, features)


def test_misaligned_pointers():
    """A kernel would fault on them."""
    odd, four = C.c_void_p(258), C.c_void_p(260)
    f = capi.lib().bsi_b200_token_logprobs
    refused(f(P, 0, 4, 64, PLAN, four, PLAN, 2, P, P, P, P, P, None))
    for i, bad in enumerate((odd, four, odd, odd, four)):
        out = [P] * 5
        out[i] = bad
        refused(f(P, 0, 4, 64, PLAN, P, PLAN, 2, *out, None))
    g, b, h = (getattr(capi.lib(), "bsi_b200_distill_" + n) for n in ("forward", "backward", "fused"))
    head = (P, 0, 4, 64, PLAN, P, P, 0, 5, 1.0, 0)
    for i in (0, 2, 4, 5):
        args = [P, 1, P, P, P, P]
        args[i] = odd
        refused(g(*head, *args, None))
    for i in (0, 2, 4):
        args = [P, P, P, 1, P, P, 64]
        args[i] = odd
        refused(b(*head, *args, None))
    for i in (0, 2, 3, 4):
        args = [P, 1, P, P, P, P, 64]
        args[i] = odd
        refused(h(*head, *args, None))
    L = capi.lib()
    refused(L.bsi_b200_fp4_quantize(P, 0, 4, 64, 64, 1, P, 32, P, odd, None))
    refused(L.bsi_b200_fp4_dequantize(P, 32, P, odd, 4, 64, 1, P, 0, 64, None))
    for i in (0, 1, 2):
        a = [P, P, P]
        a[i] = odd
        refused(L.bsi_b200_fp4_linear(P, 32, P, a[0], P, 32, P, a[1], a[2], 4, 8, 64, 1, P, 8, 0, 0, 0, None))
