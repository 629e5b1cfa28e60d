"""Token log-probabilities and distillation over the vocabulary on CPU tensors: the reference
expressions against independent ones and against differences, and the refusals."""

import math

import pytest
import torch

from ohara_b200 import ops
from ohara_b200.ops.logprobs import MAX_ALTERNATIVES, distillation_loss_reference


def test_logprobs_entropy_and_top_match_their_definitions():
    torch.manual_seed(0)
    x = torch.randn(4, 6, 33)
    tokens = torch.randint(0, 33, (4, 6))
    got = ops.token_logprobs(x, tokens, temperature=0.7, entropy=True, top=5)
    q = torch.softmax(x.double() / 0.7, dim=-1)
    torch.testing.assert_close(got.logprobs.double(), q.gather(-1, tokens[..., None])[..., 0].log(),
                               rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(got.entropy.double(), -(q * q.log()).sum(-1), rtol=1e-5, atol=1e-6)
    values, order = q.topk(5, dim=-1)
    assert torch.equal(got.top_tokens, order)
    torch.testing.assert_close(got.top_logprobs.double(), values.log(), rtol=1e-5, atol=1e-6)


def test_what_was_not_asked_for_is_none():
    x = torch.randn(3, 9)
    only_entropy = ops.token_logprobs(x, entropy=True)
    assert only_entropy.logprobs is None and only_entropy.top_tokens is None
    assert only_entropy.entropy.shape == (3,)
    assert ops.token_logprobs(x, torch.zeros(3, dtype=torch.int32)).entropy is None


def test_ties_go_to_the_lowest_index_and_padding_rows_are_empty():
    x = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 3.0], [0.0, 0.0, 0.0, 0.0, 0.0]])
    got = ops.token_logprobs(x, torch.tensor([3, -100]), entropy=True, top=4)
    assert got.top_tokens.tolist() == [[1, 2, 4, 0], [-1, -1, -1, -1]]
    assert got.logprobs.tolist() == [-math.inf, 0.0] and got.entropy[1] == 0
    assert torch.isfinite(got.entropy).all()
    assert (got.top_logprobs[1] == -math.inf).all()


def test_out_of_range_tokens_and_rows_without_a_distribution_are_nan():
    x = torch.zeros(4, 3)
    x[2] = -math.inf
    x[3, 1] = math.nan
    got = ops.token_logprobs(x, torch.tensor([3, -1, 0, 0]), entropy=True)
    assert got.logprobs.isnan().all()
    assert got.entropy.isnan().tolist() == [False, False, True, True]


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_gradients_of_logprobs_against_differences(temperature):
    torch.manual_seed(1)
    x = torch.randn(3, 11, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([4, -100, 10])

    def f(x):
        got = ops.token_logprobs(x, tokens, temperature=temperature, entropy=True, top=3)
        return got.logprobs, got.entropy, got.top_logprobs[[0, 2]]

    assert torch.autograd.gradcheck(f, (x,))


def _teacher(rows, vocab, k, dtype=torch.float32):
    scores = torch.randn(rows, vocab, dtype=dtype)
    got = torch.log_softmax(scores, -1).topk(k, dim=-1)
    return got.values, got.indices


@pytest.mark.parametrize("tail", [False, True])
def test_distillation_matches_its_definition_and_differences(tail):
    torch.manual_seed(2)
    x = torch.randn(5, 23, dtype=torch.float64, requires_grad=True)
    logp, tokens = _teacher(5, 23, 6, torch.float64)
    tokens[1, 4:] = -1
    tokens[2] = -1                       # nothing to learn from
    loss = ops.distillation_loss(x, logp, tokens, temperature=1.7, tail=tail)
    q = torch.softmax(x.detach() / 1.7, -1)
    for r in range(5):
        keep = tokens[r] >= 0
        if not keep.any():
            assert loss[r] == 0
            continue
        p = logp[r][keep].exp()
        p = p if tail else p / p.sum()
        qs = q[r][tokens[r][keep]]
        want = (p * (p / qs).log()).sum()
        if tail:
            want = want + (1 - p.sum()) * ((1 - p.sum()) / (1 - qs.sum())).log()
        torch.testing.assert_close(loss[r], want, rtol=1e-9, atol=1e-12)
    assert torch.autograd.gradcheck(
        lambda y: ops.distillation_loss(y, logp, tokens, temperature=1.7, tail=tail), (x,))


def test_distillation_edge_rows():
    x = torch.zeros(1, 6)
    # the same token twice counts with both probabilities
    twice = ops.distillation_loss(x, torch.tensor([[0.5, 0.25]]).log(), torch.tensor([[2, 2]]), tail=True)
    want = 0.5 * math.log(0.5 * 6) + 0.25 * math.log(0.25 * 6) + 0.25 * math.log(0.25 / (5 / 6))
    assert float(twice) == pytest.approx(want, rel=1e-5)
    # an entry of probability 0 adds nothing, even for a token that the student rules out
    x[0, 1] = -math.inf
    none = ops.distillation_loss(x, torch.tensor([[0.0, -math.inf]]), torch.tensor([[0, 1]]))
    assert float(none) == pytest.approx(math.log(5), rel=1e-5)
    ruled_out = ops.distillation_loss(x, torch.tensor([[0.0]]), torch.tensor([[1]]))
    assert float(ruled_out) == math.inf
    assert ops.distillation_loss(x, torch.tensor([[0.0]]), torch.tensor([[6]])).isnan().all()
    # a list that names the whole vocabulary leaves no outside mass
    logp = torch.log_softmax(torch.randn(1, 6), -1)
    whole = distillation_loss_reference(torch.randn(1, 6), logp, torch.arange(6)[None], tail=True)
    assert torch.isfinite(whole).all()


@pytest.mark.parametrize("tail", [False, True])
def test_a_teachers_top_list_feeds_the_distillation(tail):
    torch.manual_seed(3)
    teacher, student = torch.randn(7, 40), torch.randn(7, 40, requires_grad=True)
    listed = ops.token_logprobs(teacher, top=8, temperature=2.0)
    loss = ops.distillation_loss(student, listed.top_logprobs, listed.top_tokens, temperature=2.0,
                                 tail=tail)
    assert (loss > 0).all()
    same = ops.distillation_loss(teacher, listed.top_logprobs, listed.top_tokens, temperature=2.0,
                                 tail=True)
    torch.testing.assert_close(same, torch.zeros(7), rtol=0, atol=1e-5)
    loss.sum().backward()
    torch.testing.assert_close(student.grad.sum(-1), torch.zeros(7), rtol=0, atol=1e-5)


def test_linear_forms_are_the_same_functions_of_the_products():
    torch.manual_seed(4)
    hidden = torch.randn(2, 5, 16, requires_grad=True)
    weight = torch.randn(30, 16, requires_grad=True)
    tokens = torch.randint(0, 30, (2, 5))
    got = ops.linear_token_logprobs(hidden, weight, tokens, entropy=True, top=2)
    want = ops.token_logprobs(hidden @ weight.T, tokens, entropy=True, top=2)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)
    logp, ids = _teacher(10, 30, 4)
    logp, ids = logp.view(2, 5, 4), ids.view(2, 5, 4)
    loss = ops.linear_distillation_loss(hidden, weight, logp, ids, tail=True)
    torch.testing.assert_close(loss, ops.distillation_loss(hidden @ weight.T, logp, ids, tail=True))
    loss.sum().backward()
    assert hidden.grad.abs().sum() > 0 and weight.grad.abs().sum() > 0


@pytest.mark.parametrize("call,error,message", [
    (lambda x, t: ops.token_logprobs(x), ValueError, "nothing to compute"),
    (lambda x, t: ops.token_logprobs(x, t, top=8), ValueError, "top must be between"),
    (lambda x, t: ops.token_logprobs(torch.zeros(1, 4096), top=MAX_ALTERNATIVES + 1), ValueError, "top"),
    (lambda x, t: ops.token_logprobs(x, t, top=-1), ValueError, "top must be between"),
    (lambda x, t: ops.token_logprobs(x, t, temperature=0.0), ValueError, "temperature"),
    (lambda x, t: ops.token_logprobs(x, t, temperature=math.nan), ValueError, "temperature"),
    (lambda x, t: ops.token_logprobs(x, t[:2]), ValueError, "one entry per row"),
    (lambda x, t: ops.token_logprobs(x, t.float()), TypeError, "integers"),
    (lambda x, t: ops.token_logprobs(x.long(), t), TypeError, "floating point"),
    (lambda x, t: ops.token_logprobs(torch.zeros(()), entropy=True), ValueError, "vocabulary"),
    (lambda x, t: ops.token_logprobs(torch.zeros(3, 0), entropy=True), ValueError, "empty"),
    (lambda x, t: ops.distillation_loss(x, x[:, :2], t), ValueError, "entries"),
    (lambda x, t: ops.distillation_loss(x, x[:, :2], t[:, None]), ValueError, "entries"),
    (lambda x, t: ops.distillation_loss(x, x[:, :0], t[:, None][:, :0]), ValueError, "1 to"),
    (lambda x, t: ops.distillation_loss(x, x[:, :1].requires_grad_(), t[:, None]), ValueError, "detach"),
    (lambda x, t: ops.distillation_loss(x, t[:, None], t[:, None]), TypeError, "floating"),
    (lambda x, t: ops.linear_token_logprobs(x, torch.zeros(9, 6), t), ValueError, "width"),
    (lambda x, t: ops.linear_distillation_loss(x, torch.zeros(9, 7), x[:, :1], t), ValueError, "entries"),
])
def test_refusals(call, error, message):
    with pytest.raises(error, match=message):
        call(torch.zeros(3, 7), torch.zeros(3, dtype=torch.long))


def test_empty_batches():
    x = torch.zeros(0, 7)
    got = ops.token_logprobs(x, torch.zeros(0, dtype=torch.long), entropy=True, top=2)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 2)
    assert ops.distillation_loss(x, torch.zeros(0, 3), torch.zeros(0, 3, dtype=torch.long)).shape == (0,)


# -- where the framework uses them -------------------------------------------------------------------
def _tiny_llama(seed=0):
    from ohara_b200.models.llama import Config, Llama

    torch.manual_seed(seed)
    return Llama(Config(vocab_size=50, max_sequence_length=16, hidden_size=16, intermediate_size=32,
                        num_attention_heads=2, num_key_value_heads=1, num_hidden_layers=1, dropout=0.0))


def test_a_model_distils_from_another_and_gives_preference_inputs():
    from ohara_b200.dpo import dpo_loss_from_logps, linear_sequence_logps, sequence_logps

    student, teacher = _tiny_llama(0), _tiny_llama(1)
    ids = torch.randint(0, 50, (2, 9))
    x, labels = ids[:, :-1], ids[:, 1:].clone()
    labels[0, :3] = -100
    logits = student(x)
    got = student.token_logprobs(x, labels, entropy=True)
    want = torch.log_softmax(logits, -1)
    torch.testing.assert_close(got.logprobs[1], want[1].gather(-1, labels[1][:, None])[:, 0])
    assert not got.logprobs[0, :3].any() and got.entropy.shape == (2, 8)
    summed = linear_sequence_logps(student.forward_hidden(x), student.vocab_proj.weight, labels)
    torch.testing.assert_close(summed, sequence_logps(logits, labels))
    losses, _ = dpo_loss_from_logps(summed[0], summed[1], summed[0].detach(), summed[1].detach(), 0.1)
    with torch.no_grad():
        listed = teacher.token_logprobs(x, top=5, temperature=2.0)
    loss = student.distillation_loss(x, listed.top_logprobs, listed.top_tokens, temperature=2.0, tail=True)
    torch.testing.assert_close(loss, ops.distillation_loss(logits, listed.top_logprobs, listed.top_tokens,
                                                           temperature=2.0, tail=True))
    (losses + loss.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in student.parameters())


def test_a_sharded_head_is_refused():
    model = _tiny_llama()
    model.vocab_proj.weight.tensor_parallel_dim = 0
    with pytest.raises(NotImplementedError, match="vocabulary-sharded"):
        model.token_logprobs(torch.zeros(1, 2, dtype=torch.long), entropy=True)
    other = _tiny_llama()
    other._param_sharding = object()
    with pytest.raises(NotImplementedError, match="released"):
        other.distillation_loss(torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 2, 1),
                                torch.zeros(1, 2, 1, dtype=torch.long))
