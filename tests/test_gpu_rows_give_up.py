"""Waits of the kernels over rows of logits that run out: the same source with a limit that real copies miss.

A wait that gives up is an error status and NaN for the rows it touches, never an ordinary-looking number; what is under way lands
before the kernel ends, and the context stays usable."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from bsipytorch_b200 import build, bsi_ops, scoring

pytestmark = pytest.mark.gpu

SOURCE = """
#define BSI_ROWS_WAIT_CYCLES @ll
#define BSI_ROWS_WAIT_HINT 0u
#include "vocab.cu"
extern "C" int take_status() {
    int v = -1;
    return bsi::take_vocab_status(&v) == BSI_OK ? v : -1;
}
"""


class Plan(C.Structure):
    _fields_ = [("per", C.c_int64), ("block_stride", C.c_int64), ("row_stride", C.c_int64)]


# nearly every wait gives up; some do, in the middle of a CTA's rows
@pytest.fixture(scope="module", params=[0, 3500])
def impatient(request, tmp_path_factory):
    at = tmp_path_factory.mktemp("impatient")
    (at / "impatient.cu").write_text(SOURCE.replace("@", str(request.param)))
    subprocess.run(["nvcc"] + build.NVCC_FLAGS + ["-shared", "-I", build.CSRC, "-I", os.path.join(build.ROOT, "include"), "-o", str(at / "libimpatient.so"),
                    str(at / "impatient.cu"), os.path.join(build.CSRC, "common.cu")], check=True)
    lib = C.CDLL(str(at / "libimpatient.so"))
    lib.always = request.param == 0
    return lib


def p(t):
    return C.c_void_p(t.data_ptr())


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("rows,V", [(3000, 9001), (3, 50272)])
def test_scoring(impatient, rows, V):
    g = torch.Generator(device="cuda").manual_seed(rows)
    z = torch.randn(rows, V, device="cuda", generator=g) * 3
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=g)
    want = scoring.token_logprobs(z, tokens, top_k=5)
    lp, ranks, ent = torch.empty(rows, device="cuda"), torch.empty(rows, dtype=torch.long, device="cuda"), torch.empty(rows, device="cuda")
    top, ids = torch.empty(rows, 5, device="cuda"), torch.empty(rows, 5, dtype=torch.long, device="cuda")
    rc = impatient.bsi_b200_token_logprobs(p(z), C.c_int(0), C.c_int64(rows), C.c_int64(V), C.byref(Plan(0, 0, V)), p(tokens), C.byref(Plan(0, 0, 1)),
                                           C.c_int(5), p(lp), p(ranks), p(ent), p(top), p(ids), stream())
    torch.cuda.synchronize()
    lost = torch.isnan(lp)
    assert rc == 0 and impatient.take_status() == (144 if bool(lost.any()) else 0) and impatient.take_status() == 0
    assert bool(lost.any()) or not impatient.always or rows < 100        # two chunks a CTA may be there when they are first asked for
    for got, right in ((lp, want.logprobs), (ent, want.entropy), (top, want.top_logprobs)):
        assert torch.equal(torch.isnan(got).view(rows, -1).all(1), lost) and torch.equal(got[~lost], right[~lost])
    assert torch.equal(ids[~lost], want.top_ids[~lost]) and torch.equal(ranks[~lost], want.ranks[~lost])
    assert bsi_ops.device_status() == 0 and torch.equal(scoring.token_logprobs(z, tokens, top_k=5).logprobs, want.logprobs)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V", [(3000, 9001), (3, 50272)])
def test_distillation(impatient, rows, V, tail):
    g = torch.Generator(device="cuda").manual_seed(rows)
    z = torch.randn(rows, V, device="cuda", generator=g) * 3
    t, ids = torch.topk(torch.log_softmax(z + 0.5 * torch.randn(rows, V, device="cuda", generator=g), -1), 8, -1)
    weights = torch.ones(rows, device="cuda")
    weights[1::7] = 0.0
    want, want_grad = scoring.distillation_loss_and_grad(z, ids, t, 2.0, tail, weights, "none")
    each, loss, total, grad = torch.empty(rows, device="cuda"), torch.empty((), device="cuda"), torch.empty((), device="cuda"), torch.empty_like(z)
    rc = impatient.bsi_b200_distill_fused(p(z), C.c_int(0), C.c_int64(rows), C.c_int64(V), C.byref(Plan(0, 0, V)), p(ids), p(t), C.c_int(0), C.c_int(8),
                                          C.c_double(2.0), C.c_int(int(tail)), p(weights), C.c_int(0), p(each), p(loss), p(total), p(grad), C.c_int64(V),
                                          stream())
    torch.cuda.synchronize()
    lost = torch.isnan(each)
    assert rc == 0 and impatient.take_status() == (144 if bool(lost.any()) else 0)
    assert bool(lost.any()) or not impatient.always or rows < 100        # two chunks a CTA may be there when they are first asked for
    assert bool(torch.isnan(loss)) == bool(lost.any()) and not bool(lost[1::7].any())
    assert torch.equal(torch.isnan(grad).all(1), lost) and torch.equal(each[~lost], want[~lost]) and torch.equal(grad[~lost], want_grad[~lost])
    saved = torch.empty(rows, 4, device="cuda")
    rc = impatient.bsi_b200_distill_forward(p(z), C.c_int(0), C.c_int64(rows), C.c_int64(V), C.byref(Plan(0, 0, V)), p(ids), p(t), C.c_int(0), C.c_int(8),
                                            C.c_double(2.0), C.c_int(int(tail)), p(weights), C.c_int(0), p(each), p(saved), p(loss), None, stream())
    torch.cuda.synchronize()
    assert rc == 0 and impatient.take_status() == (144 if bool(torch.isnan(each).any()) else 0)
    assert torch.equal(torch.isnan(saved[:, 0]), torch.isnan(each))
    assert torch.equal(scoring.distillation_loss_and_grad(z, ids, t, 2.0, tail, weights, "none")[1], want_grad) and bsi_ops.device_status() == 0
