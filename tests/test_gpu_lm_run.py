"""The operators as they are used together: a dense model's answers, its 4-bit copy scored and distilled against them."""
import copy

import pytest
import torch

from bsipytorch_b200 import opt

pytestmark = pytest.mark.gpu

TINY = opt.OPTConfig(vocab_size=4099, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, ffn_dim=1024, max_position_embeddings=64, name="tiny")


def plain_loss(logits, ids, teacher, weights):
    """The loss with the tail as one class, in float64 by autograd's own operators."""
    logq = torch.log_softmax(logits.double(), -1)
    p = teacher.double().exp()
    rest = (1 - p.sum(-1)).clamp(min=0)
    listed = torch.zeros_like(logq, dtype=torch.bool).scatter(-1, ids, True)
    tail = torch.logsumexp(logq.masked_fill(listed, -float("inf")), -1)
    # 0 log 0 is 0: a listed probability or a rest that float32 has no room for
    each = (torch.xlogy(p, p) - p * logq.gather(-1, ids)).sum(-1) + torch.xlogy(rest, rest) - rest * tail
    return (each * weights.double()).sum() / weights.double().sum()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantise_score_distil(fmt, dtype):
    from bsipytorch_b200 import microscale, scoring
    teacher = opt.build_opt(TINY, dtype=dtype, seed=1)
    with torch.no_grad():
        teacher.lm_head.weight.mul_(8.0)                 # answers with some shape to them
    tokens = torch.randint(3, TINY.vocab_size, (3, 24), generator=torch.Generator().manual_seed(2)).cuda()
    answers = teacher.score(tokens, top_k=16)
    with torch.no_grad():
        logits = teacher(tokens)
    direct = scoring.token_logprobs(logits[:, :-1].contiguous(), tokens[:, 1:].contiguous(), 16)
    assert all(torch.equal(a, b) for a, b in zip((answers.ranks, answers.top_ids), (direct.ranks, direct.top_ids)))
    assert torch.equal(answers.top_ids[:, -1, 0], logits[:, -2].float().argmax(-1))

    student = microscale.quantize_model_fp4(copy.deepcopy(teacher), fmt, verbose=False)
    linears = [m for m in student.modules() if isinstance(m, microscale.FP4Linear)]
    assert len(linears) == 6 * TINY.num_hidden_layers
    student.requires_grad_(False)
    trained = [student.model.decoder.final_layer_norm.weight, student.model.decoder.final_layer_norm.bias]
    for p in trained:
        p.requires_grad_(True)
    weights = torch.ones(3, 23, device="cuda")
    weights[1, 10:] = 0.0

    loss = student.distillation_loss(tokens, answers.top_ids, answers.top_logprobs, tail=True, weights=weights)
    loss.backward()
    got = [p.grad.clone() for p in trained]
    for p in trained:
        p.grad = None
    logits = student(tokens)[:, :-1]
    want = plain_loss(logits, answers.top_ids, answers.top_logprobs, weights)
    (wanted,) = torch.autograd.grad(want, logits, retain_graph=True)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-4 * (1.0 + float(want.detach()))
    # the logits' gradient leaves in the logits' type, half a step off; a norm's gradient sums 59 x 4099 of them through the head
    logits.backward(wanted.to(dtype))
    for g, p in zip(got, trained):
        eps = torch.finfo(dtype).eps
        assert float((g.double() - p.grad.double()).norm()) <= (4 * eps + 1e-4) * float(p.grad.double().norm()) + 1e-7
    # the student against itself: its own answers are its own distribution
    own = student.score(tokens, top_k=16)
    with torch.no_grad():
        zero = student.distillation_loss(tokens, own.top_ids, own.top_logprobs, tail=True)
    assert abs(float(zero)) <= 2e-5
    assert float(loss.detach()) > float(zero)


def test_a_bsi_model_is_scored_too():
    model = opt.build_opt_bsi(TINY, dtype=torch.float16)
    tokens = torch.randint(3, TINY.vocab_size, (2, 16)).cuda()
    got = model.score(tokens, top_k=5)
    with torch.no_grad():
        logits = model(tokens)[:, :-1].float()
    logq = torch.log_softmax(logits, -1)
    torch.testing.assert_close(got.logprobs, logq.gather(-1, tokens[:, 1:, None])[..., 0], rtol=0, atol=2e-5)
    assert torch.equal(got.ranks == 0, logits.argmax(-1) == tokens[:, 1:])


@pytest.mark.parametrize("quantise", ["fp4", "bsi", "fp4 mlp"])
def test_what_a_quantised_student_s_gradient_reaches(quantise):
    from bsipytorch_b200 import microscale
    student = opt.build_opt_bsi(TINY, dtype=torch.float32) if quantise == "bsi" else opt.build_opt(TINY, dtype=torch.float32, seed=1)
    if quantise != "bsi":
        microscale.quantize_model_fp4(student, "nvfp4", scope="mlp" if quantise == "fp4 mlp" else "all", verbose=False)
    student.requires_grad_(True)
    tokens = torch.randint(3, TINY.vocab_size, (2, 12), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        answers = student.score(tokens, top_k=8)
    student.distillation_loss(tokens, answers.top_ids, answers.top_logprobs - 0.1, tail=True).backward()
    reached = {n for n, p in student.named_parameters() if p.grad is not None and bool(p.grad.any())}
    want = {"model.decoder.embed_tokens.weight", "model.decoder.embed_positions.weight", "model.decoder.final_layer_norm.weight",
            "model.decoder.final_layer_norm.bias"}
    if quantise == "fp4 mlp":          # the attention's projections and the norm in front of them, past the packed half of each layer
        want |= {n for n, _ in student.named_parameters() if ".self_attn." in n or ".self_attn_layer_norm." in n}
        reached |= {n for n in want if n.endswith("k_proj.bias")}      # a softmax's gradient for a shift of all its keys is 0
    assert reached == want
