"""Token log probabilities against the definition in float64."""
import numpy as np
import pytest
import torch

import _lm_oracle as oracle

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def scoring():
    from bsipytorch_b200 import scoring as m
    return m


def rows_of(kind, rows, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, V, generator=g) * 2.5
    if kind == "ties":                 # few distinct values, all of them exact in 16 bits
        z = (z * 0.8).round()
    elif kind == "constant":
        z = torch.full((rows, V), 1.5)
    elif kind == "masked":             # a constrained vocabulary: -inf nearly everywhere
        keep = torch.rand(rows, V, generator=g) < 5.0 / V
        keep[:, V // 2] = True
        z = torch.where(keep, z, torch.tensor(-float("inf")))
    elif kind == "lowest":             # the type's lowest value as a mask
        keep = torch.rand(rows, V, generator=g) < 0.5
        keep[:, V // 2] = True
        z = torch.where(keep, z, torch.tensor(torch.finfo(dtype).min))
    elif kind == "only lowest":        # nothing but the lowest value and -inf
        z = torch.where(torch.rand(rows, V, generator=g) < 0.5, torch.tensor(torch.finfo(dtype).min), torch.tensor(-float("inf")))
        z[:, V // 2] = torch.finfo(dtype).min
    elif kind == "far":                # one entry far above the rest, and levels far from zero
        z = z * 4 + 200.0
        z[:, V // 3] += 60.0
    return z.to(dtype)


# The kernel's sum of exponentials: 2^-22 for each ex2.approx, and at most 32 + V / 16384 + 25 additions behind one another (a batch,
# a thread's batches, the tree), each off by 2^-24: below 2^-24 * (4 + 32 + 13 + 25) < 5e-6 relative for V <= 200,000, so as much
# absolute on its logarithm. A log probability then rounds two float32 differences and its logarithm: 3 * 2^-24 of the terms' size.
def logprob_tolerance(logq):
    return 5e-6 + 3 * 2.0 ** -24 * (np.abs(logq) + 15.0)


# entropy = log s - ln 2 * w / s: the same error on log s (s >= 1, log s <= 13); w's terms e * d carry the same and the rounding of d,
# 3 * 2^-24 of it, and |w / s| ln 2 <= |entropy| + log s.
def entropy_tolerance(h):
    return 2 * (5e-6 + 3 * 2.0 ** -24) * (1.0 + np.abs(h) + 13.0)


def compare(z, tokens, got, k):
    zn = z.double().cpu().numpy().reshape(-1, z.shape[-1])
    tn = tokens.cpu().numpy().reshape(-1)
    lp, rank = got.logprobs.cpu().double().numpy().reshape(-1), got.ranks.cpu().numpy().reshape(-1)
    ent = got.entropy.cpu().double().numpy().reshape(-1)
    top, ids = got.top_logprobs.cpu().double().numpy().reshape(len(zn), k), got.top_ids.cpu().numpy().reshape(len(zn), k)
    for r in range(len(zn)):
        want = oracle.score(zn[r], int(tn[r]), k)
        assert rank[r] == want[1], (r, rank[r], want[1])
        assert np.array_equal(ids[r], want[4]), r
        both_inf = np.isinf(want[3]) & (top[r] == want[3])
        finite = ~both_inf
        assert np.all(np.abs(top[r][finite] - want[3][finite]) <= logprob_tolerance(want[3][finite])), r
        assert lp[r] == want[0] or abs(lp[r] - want[0]) <= logprob_tolerance(want[0]), (r, lp[r], want[0])
        assert abs(ent[r] - want[2]) <= entropy_tolerance(want[2]), (r, ent[r], want[2])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (2, 2, 2), (3, 7, 5), (5, 33, 20), (4, 130, 128), (7, 1000, 5), (2, 1027, 128),
                                      (3, 4099, 64), (1, 50272, 20), (5, 50272, 1), (2, 128011, 128), (160, 8200, 5), (300, 515, 0)])
def test_sizes(dtype, rows, V, k):
    z = rows_of("plain", rows, V, DT[dtype], rows * 31 + V)
    g = torch.Generator().manual_seed(V)
    tokens = torch.randint(0, V, (rows,), generator=g)
    tokens[0] = int(z[0].float().argmax())
    tokens[-1] = -100 if rows > 1 else tokens[-1]
    got = scoring().token_logprobs(z.cuda(), tokens.cuda(), top_k=k)
    assert got.ranks[0] == 0
    compare(z, tokens, got, k)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["ties", "constant", "masked", "lowest", "only lowest", "far"])
@pytest.mark.parametrize("rows,V,k", [(2, 300, 20), (3, 9001, 128), (1, 50272, 64)])
def test_contents(kind, dtype, rows, V, k):
    z = rows_of(kind, rows, V, DT[dtype], V)
    tokens = torch.tensor([V // 2, V - 1, 0][:rows])
    compare(z, tokens, scoring().token_logprobs(z.cuda(), tokens.cuda(), top_k=k), k)


@pytest.mark.parametrize("V", [50272, 1001])
def test_token_at_a_masked_place(V):
    z = rows_of("masked", 2, V, torch.float16, 5)
    tokens = torch.tensor([0, V - 1])
    z[:, 0] = z[:, -1] = -float("inf")
    got = scoring().token_logprobs(z.cuda(), tokens.cuda())
    assert torch.equal(got.logprobs.cpu(), torch.full((2,), -float("inf")))
    want = [oracle.score(z[r].double().numpy(), int(tokens[r]), 0)[1] for r in range(2)]
    assert got.ranks.tolist() == want


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [1003, 8192])
def test_rows_are_read_where_they_lie(dtype, V):
    """logits[:, :-1] and tokens[:, 1:] of a batch, a column slice on an odd element, a broadcast row, a transposed batch."""
    g = torch.Generator().manual_seed(3)
    whole = (torch.randn(3, 5, V + 6, generator=g) * 2).to(DT[dtype]).cuda()
    tokens = torch.randint(0, V, (3, 5), generator=g).cuda()
    m = scoring()
    for z in (whole[:, :-1, 1:V + 1], whole[:, 1:, 3:V + 3], whole.transpose(0, 1)[:3, :, :V].transpose(0, 1)):
        t = tokens[:, 1:][:, :z.shape[1]]
        compare(z, t, m.token_logprobs(z, t, top_k=7), 7)
        want = m.token_logprobs(z.contiguous(), t.contiguous(), top_k=7)
        assert all(torch.equal(a, b) for a, b in zip(want, m.token_logprobs(z.contiguous(), t, top_k=7)))
    row = whole[0, 0, :V]
    got = m.token_logprobs(row.expand(4, V), tokens.reshape(-1)[:4], top_k=3)
    compare(row.expand(4, V), tokens.reshape(-1)[:4], got, 3)
    one = m.token_logprobs(row, tokens[0, 0], top_k=3)
    assert one.logprobs.shape == () and one.top_ids.shape == (3,) and one.logprobs == got.logprobs[0]


def test_no_rows_and_no_tokens():
    m = scoring()
    got = m.token_logprobs(torch.empty(0, 11, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"), top_k=3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)
    z = torch.randn(4, 77, device="cuda")
    got = m.token_logprobs(z, top_k=2)
    assert torch.equal(got.ranks, torch.full((4,), -1, device="cuda")) and not got.logprobs.any()
    beyond = m.token_logprobs(z, torch.tensor([77, -1, 1 << 40, 3], dtype=torch.long, device="cuda"))
    assert beyond.ranks[:3].tolist() == [-1] * 3 and beyond.ranks[3] >= 0
    assert torch.equal(beyond.entropy, got.entropy)
    assert torch.equal(m.token_logprobs(z, torch.tensor([3] * 4, dtype=torch.int32, device="cuda")).ranks[3], beyond.ranks[3])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("nan")])
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_that_have_no_distribution(bad, dtype):
    z = torch.randn(3, 5000).to(DT[dtype])
    z[1, 4321] = bad
    z[2] = -float("inf")
    got = scoring().token_logprobs(z.cuda(), torch.tensor([1, 2, 3]).cuda(), top_k=4)
    for t in (got.logprobs, got.entropy):
        assert torch.isfinite(t[0]) and torch.isnan(t[1]) and torch.isnan(t[2])
    assert got.top_ids[1, 0] == 4321 and got.top_ids[2].tolist() == [0, 1, 2, 3]
    assert bool((got.top_ids >= 0).all()) and bool((got.top_ids < 5000).all())
    compare(z[:1], torch.tensor([1]), type(got)(*(t[:1] for t in got)), 4)


def test_same_bits_again_and_in_a_graph():
    z = (torch.randn(9, 50272) * 3).half().cuda()
    tokens = torch.arange(9).cuda() * 1000
    m = scoring()
    first = m.token_logprobs(z, tokens, top_k=20)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        held = m.token_logprobs(z, tokens, top_k=20)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, held))
    z.copy_((torch.randn(9, 50272) * 3).half())
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(m.token_logprobs(z, tokens, top_k=20), held))


def test_refusals():
    m = scoring()
    z = torch.randn(4, 50, device="cuda")
    ids = torch.zeros(4, dtype=torch.long, device="cuda")
    for call in (lambda: m.token_logprobs(z.cpu(), ids.cpu()), lambda: m.token_logprobs(z, ids.cpu()),
                 lambda: m.token_logprobs(z.double(), ids), lambda: m.token_logprobs(z, ids.float()),
                 lambda: m.token_logprobs(z, ids[:3]), lambda: m.token_logprobs(z, ids, top_k=51),
                 lambda: m.token_logprobs(torch.randn(2, 500, device="cuda"), top_k=129), lambda: m.token_logprobs(z, ids, top_k=-1),
                 lambda: m.token_logprobs(torch.empty(3, 0, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
