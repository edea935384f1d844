"""Distillation from a teacher's top entries: loss and gradient against the formulas in float64, and against differences."""
import numpy as np
import pytest
import torch

import _lm_oracle as oracle

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def scoring():
    from bsipytorch_b200 import scoring as m
    return m


def case(rows, V, K, dtype, tail, temperature, seed, holes=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, V, generator=g) * 2.5).to(dtype)
    t = z.float() + 0.5 * torch.randn(rows, V, generator=g)
    if tail:
        t = torch.log_softmax(t / temperature, -1)
    top, ids = torch.topk(t, K, -1)
    w = torch.rand(rows, generator=g) + 0.5
    if holes and rows > 2:
        w[1] = 0.0                          # a padded row
        ids[2, K // 2:] = -1                # a row with fewer entries
    return z, ids, top, w


# Rounding of the output, half a step of its type relative to the value. Before it, in float32: q_j = exp(x) / s has the error of s
# (5e-6 relative, see the scoring tests), of the exponent (|x| <= 40 at 3 * 2^-24 of it) and of three products; p likewise, from a
# softmax over at most 512 entries or the exponential of a given value; the factor 1 - rest / q_rest the sum of the teacher's p
# (512 additions), which enters rest as an absolute 2^-24 * 30. A gradient is a difference of q and p times a scale of at most `scale`.
def grad_tolerance(want, q_and_p, scale, dtype):
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # half a step of the type's smallest numbers
    return 1.01 * eps * np.abs(want) + tiny + scale * 2e-5 * q_and_p


def check(z, ids, t, w, temperature, tail, loss, grad, reduction="mean", upstream=1.0):
    zn, tn, wn, idn = z.double().numpy(), t.double().numpy(), w.double().numpy(), ids.numpy()
    rows, V = zn.shape
    total = wn.sum() if reduction == "mean" else 1.0
    want_loss, magnitude = [], []
    gn = grad.double().cpu().numpy()
    for r in range(rows):
        l, g = oracle.distill(zn[r], idn[r], tn[r], temperature, tail, wn[r])
        want_loss.append(l)
        q = np.exp(zn[r] / temperature - np.max(zn[r] / temperature))
        q /= q.sum()
        pq = q.copy()
        np.add.at(pq, idn[r][idn[r] >= 0], 1.0 / max(1, (idn[r] >= 0).sum()) + 1.0)      # p of a listed logit, at most about 1
        scale = abs(upstream) * wn[r] * temperature / total
        want = g * upstream / total
        far = np.abs(gn[r] - want) - grad_tolerance(want, pq, scale, z.dtype)
        assert far.max() <= 0, (r, int(far.argmax()), gn[r][far.argmax()], want[far.argmax()])
        magnitude.append(abs(l) + wn[r] * temperature ** 2 * 20.0)
    want_loss, magnitude = np.array(want_loss), np.array(magnitude)
    # each log q and log p is off by at most 1e-5 (values of up to about 40), and p by 2e-5 relative
    if reduction == "none":
        assert np.all(np.abs(loss.double().cpu().numpy() - want_loss) <= 2e-5 * magnitude)
    else:
        assert abs(float(loss) - want_loss.sum() / total) <= 2e-5 * magnitude.sum() / total


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V,K,T", [(1, 1, 1, 1.0), (3, 9, 4, 2.0), (4, 33, 33, 0.7), (5, 1000, 8, 2.0), (3, 1029, 128, 1.0),
                                        (7, 5001, 64, 3.0), (2, 50272, 64, 2.0), (3, 50275, 20, 1.0), (3, 128011, 16, 0.7),
                                        (400, 300, 5, 2.0), (3, 2000, 512, 1.0)])
def test_sizes(dtype, tail, rows, V, K, T):
    z, ids, t, w = case(rows, V, K, DT[dtype], tail, T, rows + V + K)
    m = scoring()
    args = [x.cuda() for x in (ids, t)]
    x = z.cuda().requires_grad_()
    loss = m.distillation_loss(x, *args, temperature=T, tail=tail, weights=w.cuda())
    loss.backward()
    check(z, ids, t, w, T, tail, loss.detach(), x.grad)
    both = m.distillation_loss_and_grad(z.cuda(), *args, temperature=T, tail=tail, weights=w.cuda())
    check(z, ids, t, w, T, tail, both[0], both[1])
    with torch.no_grad():
        assert torch.equal(m.distillation_loss(z.cuda(), *args, temperature=T, tail=tail, weights=w.cuda()), loss)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("tail", [False, True])
def test_reductions_and_upstream_gradients(reduction, tail):
    z, ids, t, w = case(6, 3001, 12, torch.float32, tail, 2.0, 5)
    x = z.cuda().requires_grad_()
    m = scoring()
    loss = m.distillation_loss(x, ids.cuda(), t.cuda(), 2.0, tail, w.cuda(), reduction)
    if reduction == "none":
        up = torch.linspace(-1.0, 2.0, 6)       # gradients of up to 2 w T
        (loss * up.cuda()).sum().backward()
        for r in range(6):
            l, g = oracle.distill(z[r].double().numpy(), ids[r].numpy(), t[r].double().numpy(), 2.0, tail, float(w[r]))
            assert np.abs(x.grad[r].double().cpu().numpy() - g * float(up[r])).max() <= 2e-5 * 4 * 2
            assert abs(float(loss[r].detach()) - l) <= 2e-5 * (abs(l) + 120)
    else:
        (loss * -1.75).backward()
        check(z, ids, t, w, 2.0, tail, loss.detach(), x.grad, reduction, upstream=-1.75)
    both = m.distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), 2.0, tail, w.cuda(), reduction)
    check(z, ids, t, w, 2.0, tail, both[0], both[1], reduction)


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(tail):
    """Central differences of the oracle's float64 loss pin the formula that the other tests compare with."""
    z, ids, t, w = case(3, 40, 6, torch.float32, tail, 1.7, 9)
    _, grad = scoring().distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), 1.7, tail, w.cuda(), "sum")
    h = 1e-5
    for r in range(3):
        for j in range(40):
            up, down = z[r].double().numpy().copy(), z[r].double().numpy().copy()
            up[j] += h
            down[j] -= h
            args = (ids[r].numpy(), t[r].double().numpy(), 1.7, tail, float(w[r]))
            slope = (oracle.distill(up, *args)[0] - oracle.distill(down, *args)[0]) / (2 * h)
            # differences: h^2 times a third derivative of order 1; float32 arithmetic: 2e-5 of values of up to T w = 2.6
            assert abs(float(grad[r, j]) - slope) <= 1e-8 + 2e-5 * 2.6 * 2


@pytest.mark.parametrize("tail", [False, True])
def test_an_id_listed_twice_and_ids_outside(tail):
    z, ids, t, w = case(4, 777, 8, torch.float32, tail, 1.0, 2, holes=False)
    ids[0, 5] = ids[0, 0]
    ids[1, 1:4] = ids[1, 7]
    ids[2, 0], ids[2, 3] = 777, -5
    ids[3] = -1                                   # nothing listed: no loss, no gradient
    if tail:
        t = t - 1.0                               # keeps every row's listed mass below 1
    x = z.cuda().requires_grad_()
    loss = scoring().distillation_loss(x, ids.cuda(), t.cuda(), 1.0, tail, reduction="none")
    loss.sum().backward()
    assert loss[3] == 0 and not x.grad[3].any()
    ids[2, 0] = -1
    check(z, ids, t, torch.ones(4), 1.0, tail, loss.detach(), x.grad, "none")
    both = scoring().distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), 1.0, tail, reduction="none")
    check(z, ids, t, torch.ones(4), 1.0, tail, both[0], both[1], "none")


@pytest.mark.parametrize("dtype", list(DT))
def test_masked_logits_and_whole_vocabulary_listed(dtype):
    z, ids, t, w = case(3, 64, 64, DT[dtype], True, 1.0, 4, holes=False)
    z[0, 10:20] = -float("inf")
    ids[0] = torch.where((ids[0] >= 10) & (ids[0] < 20), -1, ids[0])
    t[0] -= 0.5
    z[1, 30] = torch.finfo(DT[dtype]).min
    ids[1] = torch.where(ids[1] == 30, -1, ids[1])
    x = z.cuda().requires_grad_()
    loss = scoring().distillation_loss(x, ids.cuda(), t.cuda(), tail=True, weights=w.cuda(), reduction="none")
    loss.sum().backward()
    # row 0 and 1: the rest has to be found among logits of no probability at all, an infinite loss; row 2 is listed whole
    loss = loss.detach()
    assert torch.isfinite(loss[2]) and abs(float(loss[2]) - oracle.distill(z[2].double().numpy(), ids[2].numpy(), t[2].double().numpy(), 1.0, True, float(w[2]))[0]) <= 2e-5 * 40
    assert bool(torch.isfinite(x.grad[2]).all())
    off = scoring().distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), tail=False, weights=w.cuda())
    check(z, ids, t, w, 1.0, False, off[0], off[1])


def test_padded_rows_are_not_read_and_no_weight_at_all():
    m = scoring()
    z, ids, t, w = case(4, 2000, 8, torch.bfloat16, False, 1.0, 1)
    z[1] = float("nan")
    x = z.cuda().requires_grad_()
    loss = m.distillation_loss(x, ids.cuda(), t.cuda(), weights=w.cuda())
    loss.backward()
    assert torch.isfinite(loss) and not x.grad[1].any() and bool(torch.isfinite(x.grad).all())
    zero = torch.zeros(4, device="cuda")
    x.grad = None
    loss = m.distillation_loss(x, ids.cuda(), t.cuda(), weights=zero)
    loss.backward()
    assert loss == 0 and not x.grad.any()
    both = m.distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), weights=zero)
    assert both[0] == 0 and not both[1].any()
    none = m.distillation_loss_and_grad(z[:0].cuda(), ids[:0].cuda(), t[:0].cuda())
    assert none[0] == 0 and none[1].shape == (0, 2000)


@pytest.mark.parametrize("dtype", list(DT))
def test_slices_of_a_batch(dtype):
    m = scoring()
    g = torch.Generator().manual_seed(8)
    whole = (torch.randn(2, 4, 1011, generator=g) * 2).to(DT[dtype]).cuda()
    z = whole[:, :-1, 3:1004]
    t, ids = torch.topk(z.float() + 0.3, 9, -1)
    w = torch.rand(2, 3, generator=g).cuda()
    x = whole.clone().requires_grad_()
    loss = m.distillation_loss(x[:, :-1, 3:1004], ids, t, 2.0, weights=w)
    loss.backward()
    same = z.contiguous().requires_grad_()
    again = m.distillation_loss(same, ids, t, 2.0, weights=w)
    again.backward()
    # the pieces of a row differ with its alignment, and with them the order of its sums: the same up to rounding
    flat = z.contiguous().reshape(6, 1001).cpu(), ids.reshape(6, 9).cpu(), t.reshape(6, 9).cpu(), w.reshape(6).cpu()
    for l, gr in ((loss, x.grad[:, :-1, 3:1004]), (again, same.grad), m.distillation_loss_and_grad(z, ids, t, 2.0, weights=w)):
        check(*flat, 2.0, False, l.detach(), gr.reshape(6, 1001))
    assert not x.grad[:, -1].any() and not x.grad[..., :3].any() and not x.grad[..., 1004:].any()


def test_same_bits_and_a_captured_step():
    z, ids, t, w = (x.cuda() for x in case(40, 50272, 64, torch.bfloat16, True, 2.0, 6))
    m = scoring()

    def step(x):
        x.grad = None
        loss = m.distillation_loss(x, ids, t, 2.0, True, w)
        loss.backward()
        return loss.detach(), x.grad

    x = z.clone().requires_grad_()
    a, b = step(x), step(x)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    fused = m.distillation_loss_and_grad(z, ids, t, 2.0, True, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m.distillation_loss_and_grad(z, ids, t, 2.0, True, w)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(fused, held))


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_a_captured_training_step(reduction):
    """Forward and backward in one graph, on new logits at every replay, as a training loop that is launch-bound records them."""
    z, ids, t, w = (x.cuda() for x in case(6, 3001, 12, torch.float16, False, 2.0, 3))
    m = scoring()
    x = z.clone().requires_grad_()

    def step():
        loss = m.distillation_loss(x, ids, t, 2.0, False, w, reduction)
        (grad,) = torch.autograd.grad(loss.sum(), x)
        return loss.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (4, 5):
        with torch.no_grad():
            x.copy_(case(6, 3001, 12, torch.float16, False, 2.0, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_teacher_in_sixteen_bits_and_ids_in_32():
    z, ids, t, w = case(5, 2003, 9, torch.float32, False, 1.0, 12)
    for dtype in (torch.float16, torch.bfloat16):
        th = t.to(dtype)
        loss, grad = scoring().distillation_loss_and_grad(z.cuda(), ids.int().cuda(), th.cuda(), 1.0, False, w.cuda())
        check(z, ids, th.float(), w, 1.0, False, loss, grad)
        x = z.cuda().requires_grad_()
        scoring().distillation_loss(x, ids.int().cuda(), th.cuda(), weights=w.cuda().double()).backward()
        check(z, ids, th.float(), w, 1.0, False, loss, x.grad)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("gap", [60.0, 200.0, 5000.0, None])
def test_everything_outside_the_list_far_below(dtype, gap):
    """The student's share of what is not listed is below float32's numbers (and float64's); None: masked by the type's lowest value."""
    dt, T, K = DT[dtype], 2.0, 6
    z, ids, t, w = case(3, 1003, K, dt, True, T, 21, holes=False)
    out = torch.ones(3, 1003, dtype=torch.bool).scatter_(1, ids, False)
    z[out] = torch.finfo(dt).min if gap is None else (z.float() - gap).to(dt)[out]
    t[:] = torch.log_softmax(torch.cat([t, torch.full((3, 1), -2.0)], 1), -1)[:, :K]        # leaves a rest of some per cent
    x = z.cuda().requires_grad_()
    m = scoring()
    loss = m.distillation_loss(x, ids.cuda(), t.cuda(), T, True, w.cuda(), "none")
    loss.sum().backward()
    both = m.distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), T, True, w.cuda(), "none")
    for got_loss, got in ((loss.detach(), x.grad), (both[0], both[1])):
        for r in range(3):
            want_loss, want = oracle.distill(z[r].double().numpy(), ids[r].numpy(), t[r].double().numpy(), T, True, float(w[r]))
            # see grad_tolerance: q, p and here rest times its share of what is not listed, each 2e-5 off at most
            share = w[r].double().numpy() * T * 2e-5 * np.where(out[r].numpy(), 0.0, 3.0) + 2e-5 * np.abs(want)
            far = np.abs(got[r].double().cpu().numpy() - want) - grad_tolerance(want, 0.0, 1.0, dt) - share
            assert far.max() <= 0, (r, int(far.argmax()))
            if want_loss < 3.4e38:
                assert abs(float(got_loss[r]) - want_loss) <= 2e-5 * (abs(want_loss) + 20 * T * T * float(w[r]))


def test_autograd_s_own_rules():
    m = scoring()
    z, ids, t, w = (x.cuda() for x in case(4, 100, 5, torch.float32, False, 1.0, 1))
    x = z.clone().requires_grad_()
    loss = m.distillation_loss(x, ids, t)
    (g,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(g, torch.autograd.grad(loss, x, retain_graph=True)[0])
    with pytest.raises(RuntimeError):                     # no second derivative
        torch.autograd.grad(loss, x, create_graph=True)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError):                     # the logits were changed since
        loss.backward()
    with torch.no_grad():
        assert not m.distillation_loss(x, ids, t).requires_grad
    y = (z * 2).requires_grad_()                          # behind another operator, and in half a graph
    (m.distillation_loss(y.half() * 0.5, ids, t, weights=w) * 3).backward()
    assert y.grad.dtype == torch.float32 and torch.isfinite(y.grad).all() and y.grad.abs().sum() > 0


def test_refusals():
    m = scoring()
    z, ids, t, w = (x.cuda() for x in case(4, 100, 5, torch.float32, False, 1.0, 1))
    with pytest.raises(ValueError):
        m.distillation_loss(z, ids, t, reduction="average")
    with pytest.raises(RuntimeError):
        m.distillation_loss(z, ids, t.clone().requires_grad_())
    for call in (lambda: m.distillation_loss(z.cpu(), ids.cpu(), t.cpu()), lambda: m.distillation_loss(z, ids.float(), t),
                 lambda: m.distillation_loss(z, ids[:, :3], t), lambda: m.distillation_loss(z, ids[:3], t[:3]),
                 lambda: m.distillation_loss(z, ids, t.double()), lambda: m.distillation_loss(z, ids, t, temperature=0.0),
                 lambda: m.distillation_loss(z, ids, t, temperature=float("nan")), lambda: m.distillation_loss(z, ids, t, weights=w[:3]),
                 lambda: m.distillation_loss(z, ids, t, weights=w.cpu()), lambda: m.distillation_loss(z, ids[:, :0], t[:, :0]),
                 lambda: m.distillation_loss(z.repeat(1, 10), ids.repeat(1, 120), t.repeat(1, 120))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V", [(64, 20011), (3, 128011)])
def test_listed_entries_hold_the_mass(tail, rows, V):
    """Where q and p are both near each other and near 1 in sum, a listed entry's gradient is only as good as the row's total."""
    K = 16
    g = torch.Generator().manual_seed(V)
    z = torch.randn(rows, V, generator=g) - 30.0
    ids = torch.argsort(torch.rand(rows, V, generator=g), -1)[:, :K]
    listed = torch.randn(rows, K, generator=g)
    z.scatter_(1, ids, listed)
    t = listed + 0.3 * torch.randn(rows, K, generator=g)
    if tail:
        t = torch.log_softmax(torch.cat([t, torch.full((rows, 1), -8.0)], 1), -1)[:, :K].contiguous()
    x = z.cuda().requires_grad_()
    m = scoring()
    m.distillation_loss(x, ids.cuda(), t.cuda(), 1.0, tail, reduction="sum").backward()
    fused = m.distillation_loss_and_grad(z.cuda(), ids.cuda(), t.cuda(), 1.0, tail, reduction="sum")[1]
    # Scale 1. tail: the listed sum and the total are float64's but for the rest's share (e^-20 of it), then 1 / total, p and the
    # result are rounded once each. No tail: the total is made of ex2.approx, 2^-22 each for a term and for moving a thread's, a
    # warp's, a block's and a cluster's sum, and of K additions that are not of next to nothing.
    total = 2.0 ** -24 if tail else 5 * 2.0 ** -22 + K * 2.0 ** -24
    for got in (x.grad, fused):
        got = got.double().cpu().numpy()
        for r in range(rows):
            zn, idn = z[r].double().numpy(), ids[r].numpy()
            _, want = oracle.distill(zn, idn, t[r].double().numpy(), 1.0, tail)
            q = np.exp(zn - zn.max())
            q /= q.sum()
            p = q[idn] - want[idn]
            far = np.abs(got[r][idn] - want[idn]) - 1.02 * (total * q[idn] + 2.0 ** -24 * (p + np.abs(want[idn])))
            assert far.max() <= 0, (r, far.max(), got[r][idn][far.argmax()], want[idn][far.argmax()])
            out = np.ones(V, bool)
            out[idn] = False      # see grad_tolerance: q, and what p leaves times a logit's share of the rest, which is q's too
            assert np.all(np.abs(got[r][out] - want[out]) <= 2e-5 * (q[out] + np.abs(want[out])))


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_a_kept_loss_holds_nothing_else(reduction):
    z, ids, t, w = (x.cuda() for x in case(4096, 64, 5, torch.float32, False, 1.0, 1))
    x = z.requires_grad_()
    loss = scoring().distillation_loss(x, ids, t, weights=w, reduction=reduction)
    loss.sum().backward()
    kept = loss.detach()
    assert kept.untyped_storage().nbytes() <= kept.numel() * 4 + 511
