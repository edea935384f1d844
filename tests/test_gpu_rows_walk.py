"""Rows of logits beyond one for each CTA or cluster, and vocabularies beyond what a batch's bit or a CTA's shared memory holds.

A B200 has 592 slots of 256 threads for these kernels; with more rows a CTA goes from one to the next, its ring and its prefetches ahead of it."""
import numpy as np
import pytest
import torch

import _lm_oracle as oracle
from test_gpu_distillation import case, check, grad_tolerance
from test_gpu_scoring import compare, entropy_tolerance, logprob_tolerance, rows_of

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def scoring():
    from bsipytorch_b200 import scoring as m
    return m


def clean():
    from bsipytorch_b200 import bsi_ops
    return bsi_ops.device_status() == 0


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,V,k", [(1300, 3, 2), (1300, 515, 0), (700, 515, 5), (1300, 515, 64), (1250, 4101, 5), (700, 4101, 64), (610, 8213, 128)])
def test_scoring_walks_over_rows(dtype, rows, V, k):
    z = rows_of("plain", rows, V, DT[dtype], rows + V)
    z[::5] = rows_of("ties", rows, V, DT[dtype], 1)[::5]
    g = torch.Generator().manual_seed(V)
    tokens = torch.randint(0, V, (rows,), generator=g)
    tokens[torch.rand(rows, generator=g) < 0.2] = -100          # not scored, between rows that are
    there, ids = z.cuda(), tokens.cuda()
    got = scoring().token_logprobs(there, ids, top_k=k)
    compare(z, tokens, got, k)
    # what a row gets does not depend on the row before it: the bits of a batch whose rows have a CTA each
    if V * z.element_size() < 16384:                            # rows too short for clusters
        alone = scoring().token_logprobs(there[600:690], ids[600:690], top_k=k)
        assert all(torch.equal(a, b[600:690]) for a, b in zip(alone, got))
    assert clean()


@pytest.mark.parametrize("kind", ["plain", "ascending", "descending", "constant", "steps"])
@pytest.mark.parametrize("rows,V,k", [(1, 2200003, 20), (2, 1100001, 64), (310, 270001, 5), (300, 50003, 64)])
def test_long_rows(kind, rows, V, k):
    """Over 64 chunks of 4096 float32 a part, so that batches share a bit (the first three); rows in order, where every batch reaches the bound of its time."""
    g = torch.Generator(device="cuda").manual_seed(V)
    if kind == "plain":
        z = torch.randn(rows, V, generator=g, device="cuda") * 2.5
    elif kind == "constant":
        z = torch.full((rows, V), -3.0, device="cuda")
    else:
        z = torch.linspace(-4, 4, V, device="cuda").expand(rows, V).clone()
        if kind == "descending":
            z = z.flip(1).contiguous()
        elif kind == "steps":           # chunks in ascending order, noise within them
            z = (z * 8).floor() + torch.rand(rows, V, generator=g, device="cuda")
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
    got = scoring().token_logprobs(z, tokens, top_k=k)
    # by elementary operations in float64 on the device, a few rows at a time; more additions than the tolerances count: V / 16384 * 2^-24
    longer = V / 16384 * 2.0 ** -24
    for lo in range(0, rows, 16):
        d, t = z[lo:lo + 16].double(), tokens[lo:lo + 16, None]
        zt = d.gather(1, t)
        logq = torch.log_softmax(d, -1)
        rank = (d > zt).sum(1) + ((d == zt) & (torch.arange(V, device="cuda") < t)).sum(1)
        assert torch.equal(got.ranks[lo:lo + 16], rank)
        lp = logq.gather(1, t)[:, 0].cpu().numpy()
        assert np.all(np.abs(got.logprobs[lo:lo + 16].double().cpu().numpy() - lp) <= logprob_tolerance(lp) + longer)
        h = -(logq.exp() * logq).sum(1).cpu().numpy()
        assert np.all(np.abs(got.entropy[lo:lo + 16].double().cpu().numpy() - h) <= entropy_tolerance(h) + 2 * longer * (14.0 + np.abs(h)))
        best = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(got.top_ids[lo:lo + 16], best)
        top = logq.gather(1, best).cpu().numpy()
        assert np.all(np.abs(got.top_logprobs[lo:lo + 16].double().cpu().numpy() - top) <= logprob_tolerance(top) + longer)
    assert clean()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V,K", [(1300, 3, 2), (1300, 515, 7), (700, 4101, 64)])
def test_distillation_walks_over_rows(dtype, tail, rows, V, K):
    z, ids, t, w = case(rows, V, K, DT[dtype], tail, 2.0, rows + V)
    g = torch.Generator().manual_seed(3)
    w[torch.rand(rows, generator=g) < 0.2] = 0.0                # padded rows anywhere,
    w[100:220] = w[592 + 150:592 + 200] = 0.0                   # whole CTAs' first, second or all rows,
    w[rows - 3:] = 0.0                                          # and at the end
    w[592 + 7:592 + 9] = 1.0
    x = z.cuda().requires_grad_()
    m = scoring()
    loss = m.distillation_loss(x, ids.cuda(), t.cuda(), 2.0, tail, w.cuda())
    loss.backward()
    check(z, ids, t, w, 2.0, tail, loss.detach(), x.grad)
    both = m.distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), 2.0, tail, w.cuda())
    check(z, ids, t, w, 2.0, tail, both[0], both[1])
    each = m.distillation_loss(z.cuda(), ids.cuda(), t.cuda(), 2.0, tail, w.cuda(), "none")
    assert not each[w.cuda() == 0].any() and clean()


@pytest.mark.parametrize("rows,V", [(160, 1000003), (170, 1500001), (1, 10000001)])
def test_distillation_by_clusters_that_walk(rows, V):
    """The tail's bits: one CTA to an SM, two of them a row and 74 such pairs for 160 rows; bits that no CTA holds alone; nearly as many as a cluster holds."""
    K, T = 6, 2.0
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.empty(rows, V, dtype=torch.float16, device="cuda").normal_(0.0, 2.5, generator=g)
    ids = torch.randint(0, V, (rows, K), generator=g, device="cuda")
    z.scatter_(1, ids, 14.0)
    t = torch.log_softmax(torch.randn(rows, K + 1, generator=g, device="cuda"), -1)[:, :K].contiguous()
    w = torch.rand(rows, generator=g, device="cuda") + 0.5
    w[3:-1:4] = 0.0
    x = z.requires_grad_()
    m = scoring()
    loss = m.distillation_loss(x, ids, t, T, True, w, "none")
    loss.sum().backward()
    z = z.detach()
    both = m.distillation_loss_and_grad(z, ids, t, T, True, w, "none")
    for r in sorted({0, min(3, rows - 1), rows // 2 - 6 if rows > 20 else 0, 74 % rows, 75 % rows, rows - 2 if rows > 2 else 0, rows - 1}):
        zn, idn = z[r].double().cpu().numpy(), ids[r].cpu().numpy()
        want_loss, want = oracle.distill(zn, idn, t[r].double().cpu().numpy(), T, True, float(w[r]))
        q = np.exp((zn - zn.max()) / T)
        q /= q.sum()
        np.add.at(q, idn, 1.0 / K + 1.0)
        q *= 1.0 + V / 16384 * 2.0 ** -24 / 2e-5                 # longer sums, as below
        for l, gr in ((loss.detach(), x.grad), both):
            far = np.abs(gr[r].double().cpu().numpy() - want) - grad_tolerance(want, q, float(w[r]) * T, torch.float16)
            assert far.max() <= 0, (r, int(far.argmax()))
            # see check(): the sums are longer, V / 16384 additions of 2^-24 more
            assert abs(float(l[r]) - want_loss) <= (2e-5 + V / 16384 * 2.0 ** -24) * (abs(want_loss) + float(w[r]) * T * T * 20.0)
    assert clean()


def test_a_tail_over_more_logits_than_a_cluster_has_bits_for():
    z = torch.zeros(1, 12000000, dtype=torch.float16, device="cuda")
    ids, t = torch.zeros(1, 1, dtype=torch.long, device="cuda"), torch.full((1, 1), -1.0, device="cuda")
    with pytest.raises(RuntimeError, match="vocabulary"):
        scoring().distillation_loss(z, ids, t, tail=True)
    loss = scoring().distillation_loss(z, ids, t)                # without it any length will do: log 12000000, as p is 1
    assert abs(float(loss) - np.log(12e6)) <= (2e-5 + 12e6 / 16384 * 2.0 ** -24) * 37


def test_more_logits_than_32_bits_count():
    rows, V, K = 43001, 50003, 3                     # 2,150,179,003 of them
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda").normal_(0.0, 2.5, generator=g)
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
    got = scoring().token_logprobs(z, tokens, top_k=K)
    some = [0, rows // 2, rows - 60, rows - 1]
    compare(z[some], tokens[some], type(got)(*(t[some] for t in got)), K)
    t = got.top_logprobs + 0.1 * torch.randn(rows, K, generator=g, device="cuda")
    x = z.requires_grad_()
    scoring().distillation_loss(x, got.top_ids, t, reduction="sum").backward()
    _, grad = scoring().distillation_loss_and_grad(z.detach(), got.top_ids, t, reduction="sum")
    for gr in (x.grad, grad):
        for r in some:
            zn, idn = z[r].detach().double().cpu().numpy(), got.top_ids[r].cpu().numpy()
            want = oracle.distill(zn, idn, t[r].double().cpu().numpy(), 1.0, False)[1]
            q = np.exp(zn - zn.max())
            q /= q.sum()
            np.add.at(q, idn, 1.0 / K + 1.0)
            far = np.abs(gr[r].double().cpu().numpy() - want) - grad_tolerance(want, q, 1.0, torch.bfloat16)
            assert far.max() <= 0, (r, int(far.argmax()))
    assert clean()


@pytest.mark.parametrize("per", [0, 3, 4, 5, (1 << 31) + 1, 1 << 32, (1 << 32) + 2, 3 << 40])
def test_row_plans_of_any_number_of_rows_per_block(per):
    """C callers: 5 rows, a block of `per`; with 5 and more the block's stride says nothing."""
    import ctypes as C

    from bsipytorch_b200 import capi

    class Plan(C.Structure):
        _fields_ = [("per", C.c_int64), ("block_stride", C.c_int64), ("row_stride", C.c_int64)]

    V, K = 1001, 4
    z = torch.randn(40, V, device="cuda")
    at = [r * 2 if per in (0, 5) or per > 5 else r // per * 20 + r % per * 2 for r in range(5)]
    tokens = torch.randint(0, V, (40,), device="cuda")
    lp, top, ids = torch.empty(5, device="cuda"), torch.empty(5, K, device="cuda"), torch.empty(5, K, dtype=torch.long, device="cuda")
    plan, token_plan = Plan(per, 20 * V, 2 * V), Plan(per, 20, 2)
    capi.check(capi.lib().bsi_b200_token_logprobs(capi.ptr(z), 0, 5, V, C.byref(plan), capi.ptr(tokens), C.byref(token_plan), K, capi.ptr(lp), None, None,
                                                  capi.ptr(top), capi.ptr(ids), capi.stream_ptr()), "token_logprobs")
    want = scoring().token_logprobs(z[at], tokens[at], top_k=K)
    assert torch.equal(ids, want.top_ids)
    torch.testing.assert_close(lp, want.logprobs, rtol=0, atol=1e-5)
    each = torch.empty(5, device="cuda")
    capi.check(capi.lib().bsi_b200_distill_forward(capi.ptr(z), 0, 5, V, C.byref(plan), capi.ptr(ids), capi.ptr(top), 0, K, 1.0, 0, None, 0, capi.ptr(each),
                                                   None, None, None, capi.stream_ptr()), "distill_forward")
    torch.testing.assert_close(each, scoring().distillation_loss(z[at], ids, top, reduction="none"), rtol=0, atol=2e-5 * 20)
