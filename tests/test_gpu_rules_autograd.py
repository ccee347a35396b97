"""GPU: what token_logprob's graph keeps, and what it does not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_backward_pass_frees_what_the_call_read(cuda):
    """A loop that holds its loss until the next one holds no logits, no bias and no history with it."""
    from dvae_amd.rules import Grammar, TokenRules, token_logprob
    x = torch.randn(64, 1 << 16, device=cuda, requires_grad=True)
    b = torch.zeros(1 << 16, device=cuda, requires_grad=True)
    t, size = torch.arange(64, device=cuda), x.numel() * 4

    def loss():
        r = TokenRules(1.1, bias=b.repeat(64, 1), grammar=Grammar(torch.ones(64, 1 << 16, dtype=torch.bool, device=cuda)))
        return token_logprob(x + 1.0, t, r, torch.zeros(64, 4096, dtype=torch.int64, device=cuda),
                             state=torch.zeros(64, dtype=torch.int32, device=cuda)).sum()
    torch.autograd.grad(loss(), [x, b])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    held = loss()
    assert torch.cuda.memory_allocated() - before >= 2 * size           # logits and bias, for the backward pass
    grads = torch.autograd.grad(held, [x, b], retain_graph=True)
    again = torch.autograd.grad(held, [x, b])
    assert all(torch.equal(a, c) for a, c in zip(grads, again))
    del grads, again
    torch.cuda.synchronize()
    assert held.grad_fn is not None and torch.cuda.memory_allocated() - before < 1 << 16
    with pytest.raises(RuntimeError):                                   # a second time needs retain_graph, as everywhere
        torch.autograd.grad(held, [x, b])


def test_a_leaf_that_was_given_other_memory(cuda):
    """x.data = y after the call: the gradient is that of the values that were read."""
    from dvae_amd.rules import TokenRules, token_logprob
    g = torch.Generator().manual_seed(0)
    for vocab in (9, 700):
        first, bias = torch.randn(5, vocab, generator=g).to(cuda), torch.randn(vocab, generator=g).to(cuda)
        t = torch.tensor([0, 1, 2, 3, -1], device=cuda)
        x, b = first.clone().requires_grad_(), bias.clone().requires_grad_()
        want = torch.autograd.grad(token_logprob(x, t, TokenRules(bias=b)).sum(), [x, b])
        lp = token_logprob(x, t, TokenRules(bias=b))
        x.data, b.data = torch.zeros_like(first), torch.zeros_like(bias)
        junk = [torch.full_like(first, 7.0) for _ in range(4)] + [torch.full_like(bias, 7.0) for _ in range(4)]
        got = torch.autograd.grad(lp.sum(), [x, b])
        assert all(torch.equal(a, c) for a, c in zip(got, want)) and len(junk) == 8


@pytest.mark.parametrize("which", ["logits", "bias", "tokens"])
def test_changed_logits_bias_or_tokens_are_refused(cuda, which):
    from dvae_amd.rules import TokenRules, token_logprob
    x, b = torch.randn(3, 40, device=cuda, requires_grad=True), torch.randn(40, device=cuda, requires_grad=True)
    y, c, t = x * 2.0, b * 2.0, torch.zeros(3, dtype=torch.int64, device=cuda)
    lp = token_logprob(y, t, TokenRules(bias=c))
    with torch.no_grad():
        {"logits": y, "bias": c, "tokens": t}[which].add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        lp.sum().backward()


@pytest.mark.parametrize("temperature", [0.7, 1e-9])
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("vocab,history,dtype", [(6, 4, torch.float32), (100, 20, torch.bfloat16), (300, 0, torch.float32),
                                                 (3000, 0, torch.bfloat16), (9000, 30, torch.float32), (9001, 70000, torch.float16)])
def test_a_learned_bias_over_frozen_logits(cuda, vocab, history, dtype, per_row, temperature):
    """The bias gradient alone: the same bits as beside the logits' gradient, and no memory for that."""
    from dvae_amd.rules import TokenRules, token_logprob
    g = torch.Generator().manual_seed(vocab)
    rows = 33
    x = (torch.randn(rows, vocab, generator=g) * 2).to(dtype).to(cuda)
    b = torch.randn(*((rows,) if per_row else ()), vocab, generator=g).to(cuda).requires_grad_()
    h = torch.randint(0, vocab, (rows, history), generator=g).to(cuda) if history else None
    t, w = torch.randint(-1, vocab, (rows,), generator=g).to(cuda), torch.randn(rows, generator=g).to(cuda)
    r = TokenRules(1.2, 0.1, 0.2, b)
    y = x.clone().requires_grad_()
    want = torch.autograd.grad(token_logprob(y, t, r, h, temperature=temperature), [y, b], w)[1]
    got, = torch.autograd.grad(token_logprob(x, t, r, h, temperature=temperature), b, w)
    assert torch.equal(got, want) and torch.isfinite(got).all()
    # beside frozen logits that do have a gradient elsewhere
    part, = torch.autograd.grad(token_logprob(y, t, r, h, temperature=temperature), b, w)
    assert torch.equal(part, want)


def test_frozen_logits_cost_no_gradient(cuda):
    from dvae_amd.rules import TokenRules, token_logprob
    x = torch.zeros(256, 1 << 16, dtype=torch.bfloat16, device=cuda)
    b = torch.zeros(1 << 16, device=cuda, requires_grad=True)
    lp = token_logprob(x, torch.arange(256, device=cuda), TokenRules(bias=b)).sum()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    lp.backward()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < x.numel() * 2 and abs(float(b.grad.sum())) < 1e-3
