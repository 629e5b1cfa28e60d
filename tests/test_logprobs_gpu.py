"""The vocabulary kernels (``csrc/vocab_rows.cu``) against the reference expressions in 64 bits.

Tolerances. A kernel reads the logits exactly, so a log-probability ``l = (x - m) / T - log s`` is off
by a few roundings of its terms and by the relative error of ``s``: 2^-22 of the exponential unit, the
rounding of its argument (2 * 2^-24 * |d| for terms of weight e^-|d|, at most 2^-24 * 2 / e ...) and
one rounding per addition in a thread's chain (at most ``vocab / 512 + 16`` of them). Entropies add one
more sum of the same kind. ``_slack`` counts these in units of 2^-24. A gradient element is a sum of
terms of magnitude ``M`` (returned by the oracle), each with that relative error, rounded once to the
logits' type: half a step is ``eps / 2`` of the value, and 2^-25 absolute below fp16's normal range.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _slack(vocab: int) -> float:
    return (64 + vocab / 512) * 2.0**-24


def _close(got, want, atol, rtol, what):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    both = ~want.isnan()
    got, want = got[both], want[both]
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not got[~inf].isinf().any(), f"{what}: infinities"
    off = (got[~inf] - want[~inf]).abs() - rtol * want[~inf].abs()
    atol = atol.double()[both][~inf] if isinstance(atol, torch.Tensor) else atol
    worst = (off - atol).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} over the tolerance"


def _logits(rows, vocab, dtype, scale=3.0):
    return (scale * torch.randn(rows, vocab, device="cuda")).to(dtype)


def _oracle(x, tokens, temperature, entropy, top, grads):
    """64-bit results, gradient and the magnitude of the gradient's terms."""
    from ohara_b200.ops.logprobs import token_logprobs_reference

    wide = x.detach().double().requires_grad_()
    want = token_logprobs_reference(wide, tokens, temperature=temperature, entropy=entropy, top=top)
    outs = [t for t in want[:3] if t is not None]
    d = magnitude = None
    if grads is not None:
        d = torch.autograd.grad(outs, wide, [g.double() for g in grads])[0]
        with torch.no_grad():
            q = torch.softmax(wide / temperature, -1)
            level = torch.zeros_like(q[..., :1])
            magnitude = torch.zeros_like(q)
            todo = list(grads)
            if want.logprobs is not None:
                g = todo.pop(0).double().abs()
                level += g[..., None]
                at = tokens.clamp(0, x.shape[-1] - 1)[..., None]
                magnitude.scatter_add_(-1, at, g[..., None])
            if want.entropy is not None:
                g = todo.pop(0).double().abs()
                logq = torch.log_softmax(wide / temperature, -1).clamp_min(-1e4)
                magnitude += q * g[..., None] * (logq.abs() + want.entropy[..., None])
            if want.top_logprobs is not None:
                g = todo.pop(0).double().abs()
                level += g.sum(-1, keepdim=True)
                magnitude.scatter_add_(-1, want.top_tokens.clamp_min(0), g)
            magnitude = (magnitude + q * level) / temperature
    return want, d, magnitude


def _grad_atol(magnitude, d, dtype, vocab):
    half = torch.finfo(dtype).eps / 2
    # the exponential unit returns 0 for results below 2^-126, which a coefficient multiplies: here
    # (|g| + |g_H| (|log q| + H)) / T <= (5 + 5 (88 + 11)) / 0.25 = 2000 < 2^11, so 2^-115
    flushed = 2.0**-115
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-126
    return magnitude.nan_to_num(0.0) * 2 * _slack(vocab) + d.abs().nan_to_num(0.0) * half * 1.01 + tiny \
        + flushed


def _check(x, tokens, *, temperature=1.0, entropy=True, top=0, backward=True, leaf=None):
    """One call (on ``x``, with the gradient taken for ``leaf`` where ``x`` is a view of it)."""
    from ohara_b200 import ops

    vocab = x.shape[-1]
    source = x if leaf is None else leaf
    if backward and source.is_leaf:
        source.requires_grad_(True)
    got = ops.token_logprobs(x, tokens, temperature=temperature, entropy=entropy, top=top)
    outs = [t for t in got[:3] if t is not None]
    grads = [torch.randn_like(t) for t in outs] if backward else None
    want, d, magnitude = _oracle(x, tokens, temperature, entropy, top, grads)
    spread = 1.0 / temperature
    base = _slack(vocab) * (1 + spread)
    for name in ("logprobs", "entropy", "top_logprobs"):
        a, b = getattr(got, name), getattr(want, name)
        if b is not None:
            assert a.dtype == torch.float32 and a.shape == b.shape
            _close(a, b, base, 8 * 2.0**-24, name)
    if top:
        assert torch.equal(got.top_tokens, want.top_tokens), "top_tokens"
    if backward:
        have = torch.autograd.grad(outs, x, grads)[0]
        assert have.dtype == x.dtype and have.shape == x.shape
        _close(have, d, _grad_atol(magnitude, d, x.dtype, vocab), 0.0, "gradient")
    return got


VOCABS = [1, 2, 7, 8, 65, 512, 1000, 8191, 8193, 50257, 50304]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_logprobs_over_sizes(vocab, dtype):
    torch.manual_seed(vocab)
    for rows, top in ((1, min(20, vocab)), (5, min(1, vocab)), (67, 0)):
        x = _logits(rows, vocab, dtype)
        tokens = torch.randint(0, vocab, (rows,), device="cuda")
        tokens[3::5] = -100
        _check(x, tokens, temperature=0.8, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 50304, 128), (2, 131075, 64), (9, 50257, 20),
                                            (300, 50304, 64), (400, 1200, 128), (3, 128, 128),
                                            (40, 130, 127), (700, 9000, 5)])
def test_top_alternatives_in_order(rows, vocab, top, dtype):
    torch.manual_seed(top)
    x = _logits(rows, vocab, dtype)          # 16-bit logits tie often: ties go to the lowest index
    _check(x, None, entropy=False, top=top, backward=rows < 100)


@pytest.mark.parametrize("shape", [(3, 4, 2), (6, 7)])
def test_leading_dimensions_and_partial_queries(shape):
    torch.manual_seed(0)
    x = torch.randn(*shape, 700, device="cuda").bfloat16()
    tokens = torch.randint(0, 700, shape, device="cuda")
    _check(x, tokens, entropy=False)
    _check(x.detach(), None, entropy=True)
    _check(x.detach(), None, entropy=True, top=3)


def _layouts():
    def padded(dtype):
        leaf = torch.randn(6, 1024, device="cuda").to(dtype)
        return leaf, leaf[:, :1001]

    def shifted(dtype):  # logits[:, :-1] against labels[:, 1:], two row strides
        leaf = torch.randn(4, 9, 603, device="cuda").to(dtype)
        return leaf, leaf[:, :-1]

    def unaligned(dtype):
        leaf = torch.randn(5 * 801 + 3, device="cuda").to(dtype)
        return leaf, leaf[3:].view(5, 801)

    def transposed(dtype):
        leaf = torch.randn(640, 7, device="cuda").to(dtype)
        return leaf, leaf.t()

    def expanded(dtype):
        leaf = torch.randn(1, 3, 520, device="cuda").to(dtype)
        return leaf, leaf.expand(4, 3, 520)

    def three_strides(dtype):
        leaf = torch.randn(4, 6, 5, 530, device="cuda").to(dtype)
        return leaf, leaf[::2, ::3, ::2, 3:]

    return [padded, shifted, unaligned, transposed, expanded, three_strides]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", _layouts(), ids=lambda f: f.__name__)
def test_layouts_of_the_logits(layout, dtype):
    torch.manual_seed(1)
    leaf, x = layout(dtype)
    leaf.requires_grad_(True)
    x = layout_view(leaf, x)
    tokens = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda")
    _check(x, tokens, top=4, leaf=leaf)
    logp, ids = _list_of(x.shape[:-1], x.shape[-1], 5)
    _check_distill(x, logp, ids, tail=True, leaf=leaf)


def layout_view(leaf, like):
    """The same view of ``leaf``, made after it began to require a gradient."""
    return leaf.as_strided(like.shape, like.stride(), like.storage_offset())


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_special_logits(dtype):
    torch.manual_seed(2)
    vocab = 3001
    x = _logits(12, vocab, dtype)
    low = torch.finfo(dtype).min
    x[0, 5:] = -math.inf                      # a handful of tokens left
    x[1] = low                                # everything at the type's lowest value
    x[2, ::2] = low
    x[3] = -math.inf
    x[3, 77] = 1.0                            # one token left
    x[4] = -math.inf                          # nothing left
    x[5, 9] = math.nan
    x[6, 10] = math.inf
    x[7] = 0.0
    x[7, ::3] = -0.0                          # equal to +0
    x[8] = torch.finfo(dtype).max
    x[9, 3] = torch.finfo(dtype).max
    tokens = torch.randint(0, 5, (12,), device="cuda")
    got = _check(x, tokens, top=40, backward=False)
    assert torch.equal(got.top_tokens[7], torch.arange(40, device="cuda"))
    assert got.top_tokens[5, 0] == 9 and got.top_tokens[6, 0] == 10
    keep = [0, 1, 2, 3, 7, 8, 9, 10, 11]
    for temperature in (0.25, 1.0, 30.0):
        _check(x[keep].detach(), tokens[keep], temperature=temperature, top=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top", [(50304, 128), (50257, 20), (9001, 128), (4100, 3)])
def test_rows_that_defeat_the_candidate_bound(vocab, top, dtype):
    """Constant rows, rows in ascending and descending order, and all large values in one place."""
    ramp = torch.arange(vocab, device="cuda", dtype=torch.float32)
    block = torch.zeros(vocab, device="cuda")
    block[1000:1000 + 3000] = torch.linspace(3, 5, 3000, device="cuda")
    x = torch.stack([torch.zeros(vocab, device="cuda"), ramp * 2.0**-10, -ramp * 2.0**-10, block,
                     torch.full((vocab,), -math.inf, device="cuda"), (ramp * 37) % 101])
    x[4, vocab - 2:] = 1.0
    for repeat in (1, 80, 170):               # a cluster per row; blocks of 256 and of 128 threads
        _check(x.to(dtype).repeat(repeat, 1), None, entropy=False, top=top, backward=False)


def test_tokens_outside_the_vocabulary():
    from ohara_b200 import ops

    x = _logits(5, 600, torch.float32).requires_grad_()
    tokens = torch.tensor([0, 600, -1, -100, 2**40], device="cuda")
    got = ops.token_logprobs(x, tokens, entropy=True)
    assert got.logprobs.isnan().tolist() == [False, True, True, False, True]
    assert torch.isfinite(got.entropy).all()
    (d,) = torch.autograd.grad(got.logprobs, x, torch.ones(5, device="cuda"))
    assert d.isnan().all(dim=1).tolist() == [False, True, True, False, True]
    assert (d[3] == 0).all()
    logp = torch.full((2, 2), math.log(0.4), device="cuda")
    ids = torch.tensor([[1, 600], [1, 2]], device="cuda")
    x2 = x[:2].detach().requires_grad_()
    loss = ops.distillation_loss(x2, logp, ids)
    assert loss.isnan().tolist() == [True, False]
    (d,) = torch.autograd.grad(loss.sum(), x2)
    assert d.isnan().all(dim=1).tolist() == [True, False]


def test_rows_without_an_incoming_gradient_get_zeros():
    from ohara_b200 import ops

    x = _logits(4, 700, torch.bfloat16)
    x[1, 3] = math.nan
    x.requires_grad_()
    got = ops.token_logprobs(x, torch.zeros(4, dtype=torch.long, device="cuda"), entropy=True, top=2)
    (d,) = torch.autograd.grad([got.logprobs, got.top_logprobs], x,
                               [torch.tensor([1.0, 0, 0, 2], device="cuda"),
                                torch.tensor([[0.0, 0], [0, 0], [1, 0], [0, 0]], device="cuda")])
    assert (d[1] == 0).all() and torch.isfinite(d).all() and (d[[0, 2, 3]] != 0).any(dim=1).all()


# -- distillation ------------------------------------------------------------------------------------
def _list_of(lead, vocab, k):
    scores = torch.randn(*lead, k + 1, device="cuda") * 2
    logp = torch.log_softmax(scores, -1)[..., :-1].contiguous()
    ids = torch.rand(*lead, vocab, device="cuda").topk(k, dim=-1).indices
    return logp, ids


def _check_distill(x, logp, ids, *, tail, temperature=1.0, leaf=None):
    from ohara_b200 import ops
    from ohara_b200.ops.logprobs import distillation_loss_reference

    vocab = x.shape[-1]
    if leaf is None:
        x.requires_grad_(True)
    loss = ops.distillation_loss(x, logp, ids, temperature=temperature, tail=tail)
    assert loss.dtype == torch.float32 and loss.shape == x.shape[:-1]
    wide = x.detach().double().requires_grad_()
    want = distillation_loss_reference(wide, logp.double(), ids, temperature=temperature, tail=tail)
    # a sum of K products of O(log-probability) terms, each with the error of a log-probability, and
    # 1 - sum p, off by (K + 2) 2^-24, in front of a logarithm of at most log(1e6) + 16
    k = ids.shape[-1]
    atol = 2 * _slack(vocab) * (1 + 1 / temperature) + (k + 2) * 2.0**-24 * (30 if tail else 4)
    _close(loss, want, atol, 16 * 2.0**-24, "loss")
    g = torch.rand_like(loss) + 0.5
    (have,) = torch.autograd.grad(loss, x, g)
    (d,) = torch.autograd.grad(want, wide, g.double())
    with torch.no_grad():
        q = torch.softmax(wide / temperature, -1)
        p = logp.double().masked_fill(ids < 0, -math.inf)
        p = p.exp() if tail else torch.softmax(p, -1).nan_to_num(0.0)
        magnitude = torch.zeros_like(q).scatter_add_(-1, ids.clamp(0, vocab - 1), p)
        magnitude = (magnitude + 2 * q + (k * q if tail else 0)) * g.double()[..., None] / temperature
        if tail:  # p' / q' multiplies q: its relative error is that of p', (K + 2) 2^-24 / p'
            rest = (1 - p.sum(-1)).clamp_min(1e-6)
            outside = (1 - torch.zeros_like(q).scatter_(-1, ids.clamp(0, vocab - 1),
                                                        q.gather(-1, ids.clamp(0, vocab - 1)))
                       .sum(-1)).clamp_min(1e-12)
            magnitude += q * (g.double() / temperature * (rest + (k + 2) / 64) / outside)[..., None]
    _close(have, d, _grad_atol(magnitude, d, x.dtype, vocab), 0.0, "gradient")
    return loss


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,k", [(1, 50304, 32), (3, 50257, 128), (400, 1003, 7), (6, 9, 3),
                                          (320, 20001, 16), (2, 131075, 64), (5, 2, 1)])
def test_distillation_over_sizes(rows, vocab, k, tail, dtype):
    torch.manual_seed(k)
    x = _logits(rows, vocab, dtype)
    logp, ids = _list_of((rows,), vocab, k)
    if k > 2:
        ids[::3, k - 1:] = -1
        logp[1::3, 0] = -math.inf
    if rows > 2:
        ids[2] = -1
    _check_distill(x, logp, ids, tail=tail, temperature=1.3)


@pytest.mark.parametrize("tail", [False, True])
def test_distillation_of_repeated_and_edge_tokens(tail):
    torch.manual_seed(5)
    leaf = torch.randn(4 * 515 + 1, device="cuda").requires_grad_()
    x = leaf[1:].view(4, 515)             # rows with heads and tails around the 16-byte vectors
    ids = torch.tensor([[0, 1, 2, 514], [513, 514, 512, 0], [3, 3, 3, 3], [7, 8, 7, 9]], device="cuda")
    logp = torch.log(torch.tensor([[0.3, 0.2, 0.1, 0.2]], device="cuda")).expand(4, 4)
    _check_distill(x, logp, ids, tail=tail, leaf=leaf)


def test_distillation_where_the_student_rules_tokens_out():
    from ohara_b200 import ops

    x = _logits(5, 900, torch.float32)
    x[0, 4] = -math.inf                       # a listed token: infinite
    x[1, 5:] = -math.inf                      # everything outside the list, which leaves mass there
    x[2, 5:] = -math.inf                      # the same under a list without mass outside
    x[3, 4] = -math.inf                       # listed with probability 0
    ids = torch.arange(5, device="cuda").expand(5, 5).contiguous()
    logp = torch.log(torch.tensor([0.2, 0.2, 0.2, 0.1, 0.1], device="cuda")).repeat(5, 1)
    logp[2] = torch.log_softmax(torch.randn(5, device="cuda"), -1)
    logp[3, 4] = -math.inf
    x.requires_grad_()
    loss = ops.distillation_loss(x, logp, ids, tail=True)
    assert loss.isinf().tolist() == [True, True, False, False, False]
    assert not loss.isnan().any()
    (d,) = torch.autograd.grad(loss[[2, 3, 4]].sum(), x)
    assert torch.isfinite(d).all() and (d[[0, 1]] == 0).all()


# -- from hidden states --------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width,vocab", [(1, 64, 520), (37, 256, 1003), (300, 128, 8192), (1029, 768, 5000)])
@pytest.mark.parametrize("which", ["logprobs", "renormalised", "tail"])
def test_linear_forms(rows, width, vocab, which):
    """Logits are exact products summed in fp32 (``width`` additions of terms of size |h||w|), the
    chunk's gradient is rounded to bf16 (2^-9 of each element, independent), results to bf16."""
    from ohara_b200 import ops
    from ohara_b200.ops.logprobs import distillation_loss_reference, token_logprobs_reference

    torch.manual_seed(rows)
    hidden = torch.randn(rows, width, device="cuda").bfloat16().requires_grad_()
    weight = (2 * torch.randn(vocab, width, device="cuda") / width**0.5).bfloat16().requires_grad_()
    wide = [t.detach().double().requires_grad_() for t in (hidden, weight)]
    logits = wide[0] @ wide[1].T
    if which == "logprobs":
        tokens = torch.randint(0, vocab, (rows,), device="cuda")
        tokens[1::4] = -100
        got = ops.linear_token_logprobs(hidden, weight, tokens, temperature=0.9, entropy=True)
        want = token_logprobs_reference(logits, tokens, temperature=0.9, entropy=True)
        got, want = list(got[:2]), list(want[:2])
    else:
        logp, ids = _list_of((rows,), vocab, 6)
        tail = which == "tail"
        got = [ops.linear_distillation_loss(hidden, weight, logp, ids, tail=tail)]
        want = [distillation_loss_reference(logits, logp.double(), ids, tail=tail)]
    terms = (wide[0].detach().abs() @ wide[1].detach().abs().T).max().item()
    for a, b in zip(got, want):
        # sums of `width` terms: rounding errors add up like a walk, 8 of its widths
        _close(a, b, 4 * _slack(vocab) + 8 * terms * width**0.5 * 2.0**-24, 16 * 2.0**-24, which)
    g = [torch.rand_like(t) + 0.5 for t in got]
    have = torch.autograd.grad(got, [hidden, weight], g)
    ref = torch.autograd.grad(want, wide, [t.double() for t in g])
    for a, b, name in zip(have, ref, ("d_hidden", "d_weight")):
        # each of the products' terms and each result is off by 2^-9 at most, on average less: a
        # norm error of two such roundings
        off = (a.double() - b).norm() / b.norm()
        assert off < 2 * 2.0**-9 * 1.1, f"{name}: {off}"


@pytest.mark.parametrize("top", [0, 3])
def test_linear_form_over_several_chunks_and_fp32_masters(monkeypatch, top):
    from ohara_b200 import ops
    from ohara_b200.ops import logprobs

    torch.manual_seed(7)
    hidden = torch.randn(2, 333, 128, device="cuda").requires_grad_()
    weight = (0.2 * torch.randn(777, 128, device="cuda")).requires_grad_()
    tokens = torch.randint(0, 777, (2, 333), device="cuda")

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            got = ops.linear_token_logprobs(hidden, weight, tokens, entropy=True, top=top)
        grads = torch.autograd.grad([got.logprobs, got.entropy], [hidden, weight],
                                    [torch.ones_like(got.logprobs), torch.ones_like(got.entropy)])
        return got, grads

    whole, whole_grads = run()
    monkeypatch.setattr(logprobs, "_CHUNK_BYTES", 1)   # 256 rows at a time
    parts, part_grads = run()
    # how a row is cut over threads depends on the number of rows: each side is off by a slack
    assert top == 0 or torch.equal(whole.top_tokens, parts.top_tokens)
    torch.testing.assert_close(parts.logprobs, whole.logprobs, rtol=16 * 2.0**-24,
                               atol=4 * _slack(777))
    assert whole_grads[0].dtype == torch.float32 and whole_grads[1].dtype == torch.float32
    for a, b in zip(part_grads, whole_grads):  # bf16 roundings of the logits' gradient may differ
        assert (a - b).norm() / b.norm() < 2 * 2.0**-9


# -- how they are called ---------------------------------------------------------------------------------
def test_a_teachers_list_and_the_distillation_together():
    """Write the teacher's list, distill from it with the hidden-state form, keep the policy's
    log-probabilities of the same batch: the three as one step uses them."""
    from ohara_b200 import ops

    torch.manual_seed(8)
    b, t, width, vocab = 2, 65, 128, 1003
    hidden = torch.randn(b, t, width, device="cuda").bfloat16().requires_grad_()
    weight = (2 * torch.randn(vocab, width, device="cuda") / width**0.5).bfloat16().requires_grad_()
    labels = torch.randint(0, vocab, (b, t), device="cuda")
    labels[0, :20] = -100
    with torch.no_grad():
        teacher = 2 * torch.randn(b, t, vocab, device="cuda").bfloat16()
        listed = ops.token_logprobs(teacher[:, :-1], labels[:, 1:], top=16, temperature=2.0)
    loss = ops.linear_distillation_loss(hidden[:, :-1], weight, listed.top_logprobs,
                                        listed.top_tokens, temperature=2.0, tail=True)
    assert (loss[0, :19] == 0).all() and (loss[1] > 0).all()
    policy = ops.linear_token_logprobs(hidden[:, :-1], weight, labels[:, 1:])
    total = loss.sum() * 4.0 - policy.logprobs.sum()
    d_hidden, d_weight = torch.autograd.grad(total, [hidden, weight])
    assert (d_hidden[0, :19] == 0).all() and (d_hidden[:, -1] == 0).all()
    wide = [x.detach().double().requires_grad_() for x in (hidden, weight)]
    logits = wide[0][:, :-1] @ wide[1].T
    from ohara_b200.ops.logprobs import distillation_loss_reference, token_logprobs_reference

    ref = 4 * distillation_loss_reference(logits, listed.top_logprobs.double(), listed.top_tokens,
                                          temperature=2.0, tail=True).sum()
    ref = ref - token_logprobs_reference(logits, labels[:, 1:]).logprobs.sum()
    assert abs(total.item() - ref.item()) < 1e-5 * abs(ref.item())
    for a, w in zip((d_hidden, d_weight), torch.autograd.grad(ref, wide)):
        assert (a.double() - w).norm() / w.norm() < 3 * 2.0**-9


def test_the_same_bits_every_time():
    from ohara_b200 import ops

    torch.manual_seed(9)
    x = _logits(300, 5003, torch.bfloat16).requires_grad_()
    tokens = torch.randint(0, 5003, (300,), device="cuda")
    logp, ids = _list_of((300,), 5003, 16)
    ids[:, 3] = ids[:, 5]

    def step():
        got = ops.token_logprobs(x, tokens, entropy=True, top=64)
        loss = ops.distillation_loss(x, logp, ids, tail=True)
        d = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs, loss], x,
                                [torch.ones_like(t) for t in (*got[:3], loss)])
        return [*got, loss, *d]

    first = [t.clone() for t in step()]
    blocks = [torch.full((n,), math.nan, device="cuda") for n in (300, 1200, 300 * 64, 300 * 5003 // 2)]
    del blocks
    for a, b in zip(first, step()):
        assert torch.equal(a, b)


def test_another_stream_and_two_captured_graphs():
    from ohara_b200 import ops

    torch.manual_seed(10)
    x = _logits(3, 50304, torch.bfloat16)
    tokens = torch.randint(0, 50304, (3,), device="cuda")
    want = ops.token_logprobs(x, tokens, entropy=True, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.token_logprobs(x, tokens, entropy=True, top=20)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)

    graphs, outs, inputs = [], [], []
    ids, grad = torch.arange(4, device="cuda"), torch.ones(4, device="cuda")
    for _ in range(2):
        buf = _logits(4, 50304, torch.bfloat16).requires_grad_()
        inputs.append(buf)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.token_logprobs(buf, ids, entropy=True, top=8)
            d = torch.autograd.grad(got.logprobs, buf, grad)[0]
        graphs.append(graph)
        outs.append([t.detach() for t in (*got, d)])
    for attempt in range(2):
        fresh = [_logits(4, 50304, torch.bfloat16) for _ in graphs]
        for buf, new in zip(inputs, fresh):
            buf.data.copy_(new)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):   # both in flight at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for new, out in zip(fresh, outs):
            new.requires_grad_()
            again = ops.token_logprobs(new, torch.arange(4, device="cuda"), entropy=True, top=8)
            d = torch.autograd.grad(again.logprobs, new, torch.ones(4, device="cuda"))[0]
            for a, b in zip(out, (*again, d)):
                assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Row 4100 of a 2^19-token bf16 matrix begins past 2^31 elements and 2^32 bytes."""
    from ohara_b200 import ops

    rows, vocab = 4100, 1 << 19
    if torch.cuda.mem_get_info()[0] < 14e9:
        pytest.skip("needs 14 GB of device memory")
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(3, vocab, device="cuda").bfloat16()
    x[-3:] = last
    tokens = torch.full((rows,), -100, device="cuda")
    tokens[-3:] = torch.tensor([5, vocab - 1, 77], device="cuda")
    x.requires_grad_()
    got = ops.token_logprobs(x, tokens, top=4)
    alone = last.clone().requires_grad_()
    want = ops.token_logprobs(alone, tokens[-3:], top=4)
    # the same rows alone run as clusters: the sums are taken in another order
    torch.testing.assert_close(got.logprobs[-3:], want.logprobs, rtol=0, atol=2 * _slack(vocab))
    assert torch.equal(got.top_tokens[-3:], want.top_tokens)
    g = torch.ones(rows, device="cuda")
    (d,) = torch.autograd.grad(got.logprobs, x, g)
    (dw,) = torch.autograd.grad(want.logprobs, alone, g[-3:])
    torch.testing.assert_close(d[-3:].float(), dw.float(), rtol=2.0**-7, atol=0)
    assert not d[:100].any() and not d[-100:-3].any()


def test_refusals_on_cuda():
    from ohara_b200 import ops

    x = torch.zeros(3, 9, device="cuda")
    with pytest.raises(TypeError, match="float32"):
        ops.token_logprobs(x.double(), entropy=True)
    with pytest.raises(ValueError, match="device"):
        ops.token_logprobs(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="device"):
        ops.distillation_loss(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.long))
    with pytest.raises(ValueError, match="device"):
        ops.linear_token_logprobs(x.bfloat16(), torch.zeros(4, 9), entropy=True)
    got = ops.token_logprobs(x.requires_grad_(), entropy=True)
    (d,) = torch.autograd.grad(got.entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    empty = ops.token_logprobs(torch.zeros(0, 9, device="cuda"), entropy=True, top=2)
    assert empty.entropy.shape == (0,) and empty.top_tokens.shape == (0, 2)
    none = ops.linear_token_logprobs(torch.zeros(0, 16, device="cuda").bfloat16(),
                                     torch.zeros(9, 16, device="cuda").bfloat16(), entropy=True)
    assert none.entropy.shape == (0,)


@pytest.mark.parametrize("rows,width,vocab", [(3, 8, 1), (5, 24, 7), (2, 8, 257), (257, 72, 300), (129, 1096, 129)])
@pytest.mark.parametrize("tail", [False, True])
def test_linear_forms_at_edge_sizes(rows, width, vocab, tail):
    """One-token vocabularies, widths below and beside the 64-wide steps, one row past a tile."""
    from ohara_b200 import ops
    from ohara_b200.ops.logprobs import distillation_loss_reference, token_logprobs_reference

    torch.manual_seed(vocab)
    hidden = torch.randn(rows, width, device="cuda").bfloat16().requires_grad_()
    weight = (2 * torch.randn(vocab, width, device="cuda") / width**0.5).bfloat16().requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    k = min(3, vocab)
    logp, ids = _list_of((rows,), vocab, k)
    ids[0] = -1
    wide = [t.detach().double().requires_grad_() for t in (hidden, weight)]
    logits = wide[0] @ wide[1].T
    got = ops.linear_token_logprobs(hidden, weight, tokens, entropy=True)
    loss = ops.linear_distillation_loss(hidden, weight, logp, ids, tail=tail)
    want = token_logprobs_reference(logits, tokens, entropy=True)
    ref = distillation_loss_reference(logits, logp.double(), ids, tail=tail)
    terms = (wide[0].detach().abs() @ wide[1].detach().abs().T).max().item()
    atol = 4 * _slack(vocab) + 8 * terms * width**0.5 * 2.0**-24
    _close(got.logprobs, want.logprobs, atol, 16 * 2.0**-24, "logprobs")
    _close(got.entropy, want.entropy, 2 * atol, 16 * 2.0**-24, "entropy")
    _close(loss, ref, 2 * atol + 40 * (k + 2) * 2.0**-24, 16 * 2.0**-24, "loss")
    have = torch.autograd.grad([got.logprobs, loss], [hidden, weight], [torch.ones_like(loss)] * 2)
    wanted = torch.autograd.grad([want.logprobs, ref], wide, [torch.ones_like(ref)] * 2)
    for a, b in zip(have, wanted):
        # two operators' gradients, each rounded to bf16 with its inputs, and their sum: 3 roundings of
        # magnitudes that the sum may cancel, so against the larger of the parts
        assert (a.double() - b).norm() <= 6 * 2.0**-9 * max(b.norm(), 0.05 * rows**0.5)


def test_linear_gradients_one_at_a_time_and_of_nothing():
    from ohara_b200 import ops

    torch.manual_seed(11)
    hidden = torch.randn(2, 40, 64, device="cuda").bfloat16()
    weight = torch.randn(600, 64, device="cuda").bfloat16()
    tokens = torch.randint(0, 600, (2, 40), device="cuda", dtype=torch.int32)

    def grads(h, w):
        leaves = [t for t in (h, w) if t.requires_grad]
        got = ops.linear_token_logprobs(h, w, tokens, ignore_index=7)
        return torch.autograd.grad(got.logprobs.sum(), leaves)

    both = grads(hidden.clone().requires_grad_(), weight.clone().requires_grad_())
    (only_h,) = grads(hidden.clone().requires_grad_(), weight)
    (only_w,) = grads(hidden, weight.clone().requires_grad_())
    assert torch.equal(both[0], only_h) and torch.equal(both[1], only_w)
    # rows that are strided, expanded or not aligned are laid out for the product first
    wide = torch.randn(40, 80, device="cuda").bfloat16()
    for h in (wide[:, 3:67], wide[:, :64], wide[:1, :64].expand(40, 64), wide.t()[:64].t()):
        got = ops.linear_token_logprobs(h, weight, tokens[0])
        want = ops.linear_token_logprobs(h.contiguous(), weight, tokens[0])
        assert torch.equal(got.logprobs, want.logprobs)
    none = torch.zeros(0, 64, device="cuda").bfloat16().requires_grad_()
    w = weight.clone().requires_grad_()
    loss = ops.linear_distillation_loss(none, w, torch.zeros(0, 2, device="cuda"),
                                        torch.zeros(0, 2, device="cuda", dtype=torch.long))
    d_none, d_w = torch.autograd.grad(loss.sum(), [none, w])
    assert d_none.shape == (0, 64) and not d_w.any()


def test_hidden_state_forms_captured_and_replayed():
    from ohara_b200 import ops

    torch.manual_seed(12)
    weight = torch.randn(1003, 128, device="cuda").bfloat16().requires_grad_()
    hidden = torch.randn(33, 128, device="cuda").bfloat16().requires_grad_()
    tokens = torch.randint(0, 1003, (33,), device="cuda")
    logp, ids = _list_of((33,), 1003, 5)
    g = torch.ones(33, device="cuda")

    def step(h):
        got = ops.linear_token_logprobs(h, weight, tokens, entropy=True)
        loss = ops.linear_distillation_loss(h, weight, logp, ids, tail=True)
        return (got.logprobs, got.entropy, loss,
                *torch.autograd.grad([got.logprobs, got.entropy, loss], [h, weight], [g, g, g]))

    step(hidden)                                  # sets the kernels up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [t.detach() for t in step(hidden)]   # no autograd graph outlives the capture
    for _ in range(2):
        fresh = torch.randn(33, 128, device="cuda").bfloat16()
        hidden.data.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(fresh.requires_grad_())):
            assert torch.equal(a, b)


def test_gradient_keeps_the_layout_of_a_padded_vocabulary():
    from ohara_b200 import ops

    leaf = torch.randn(6, 1024, device="cuda").bfloat16().requires_grad_()
    x = leaf[:, :1001]
    got = ops.token_logprobs(x, torch.zeros(6, dtype=torch.long, device="cuda"))
    (d,) = torch.autograd.grad(got.logprobs.sum(), x, retain_graph=True)
    assert d.stride() == x.stride() and d.shape == x.shape
    (whole,) = torch.autograd.grad(got.logprobs.sum(), leaf)
    assert torch.equal(whole[:, :1001], d) and not whole[:, 1001:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_top_list_of_a_vocabulary_beyond_the_short_positions(dtype):
    """Past 2^19 16-bit logits a vector's position no longer fits the short code: ties, masked rows."""
    torch.manual_seed(13)
    vocab = 1_200_003
    x = _logits(3, vocab, dtype)
    x[1, 50:] = -math.inf
    x[2] = 0.25
    for repeat in (1, 100):
        _check(x.repeat(repeat, 1), None, entropy=False, top=100, backward=False)


def test_tail_marks_of_a_large_vocabulary():
    from ohara_b200 import ops

    torch.manual_seed(14)
    rows, vocab = 297, 300_001                # 75 KB of marks per block
    x = _logits(rows, vocab, torch.float32)
    scores = torch.log_softmax(torch.randn(rows, 9, device="cuda"), -1)[:, :-1].contiguous()
    ids = torch.randint(0, vocab, (rows, 8), device="cuda")
    ids[:, 0] = vocab - 1
    _check_distill(x, scores, ids, tail=True)
    # more marks than a block has room for: refused before anything is launched
    huge = torch.zeros(1, 1_700_000, device="cuda").bfloat16().expand(rows, -1)
    with pytest.raises(RuntimeError, match="too large"):
        ops.distillation_loss(huge, scores, ids, tail=True)
    assert torch.isfinite(ops.distillation_loss(huge, scores, ids)).all()


def test_a_single_row_without_leading_dimensions():
    from ohara_b200 import ops

    x = torch.randn(300, device="cuda", requires_grad=True)
    token = torch.tensor(7, device="cuda")
    got = _check(x, token, top=3)
    assert got.logprobs.shape == () and got.top_tokens.shape == (3,)
    _check_distill(x, *_list_of((), 300, 4), tail=True)
    hidden = torch.randn(64, device="cuda").bfloat16().requires_grad_()
    weight = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
    alone = ops.linear_token_logprobs(hidden, weight, token, entropy=True)
    d = torch.autograd.grad([alone.logprobs, alone.entropy], [hidden, weight])
    rows = hidden.detach()[None].clone().requires_grad_()
    batch = ops.linear_token_logprobs(rows, weight, token[None], entropy=True)
    e = torch.autograd.grad([batch.logprobs.sum(), batch.entropy.sum()], [rows, weight])
    assert alone.logprobs.shape == () and torch.equal(alone.logprobs, batch.logprobs[0])
    assert torch.equal(d[0], e[0][0]) and torch.equal(d[1], e[1])
