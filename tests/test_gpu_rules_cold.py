"""GPU: token rules at low temperatures, where the part of a value that fp32 drops decides -- against oracle/rules_ref.py.

Values there are doubles: y of the kernel and of the oracle are sums, products and quotients of the same doubles in the same
order (x rho, x / rho, - frequency c, - presence, + bias: 5 roundings, the kernel's division off by one step more), so they differ by
at most 6 steps of 2^-52 relative to the largest intermediate value A: E = 6 2^-52 A.  An exponent (y - top) / T is then off by 2 E / T plus
3 roundings of a double, log Z by no more than the exponents of the weights that matter.
* log p: 4 E / T + 2^-24 |log p| (one rounding to fp32) + 1e-11 (exp2 and log of the kernel).
* gradients g / T ([v = t] - p) times the slope: p off by p (4 E / T + 1e-11), the difference rounded to fp32, then times the
  slope's rounding, the product's, and the one to the type.
Where |x4| / T is ordinary (below 277), sums over more than 128 tokens are fp32 ones: the bounds of test_gpu_rules.py."""
import math

import numpy as np
import pytest
import torch

from oracle import rules_ref as R
from test_gpu_rules import TINY, TYPES, U, half, log_z_tol, same_or_close

pytestmark = pytest.mark.gpu

COLD = [1e-2, 1e-4, 1e-6, 1e-9, 1e-10, 1e-37]


class Cold:
    """Rows whose largest values lie between two floats: 0, 1 a counted token on top (7.3 / 1.3 lies below its float, 13.7 / 1.3
    above); 2 a biased one; 3, 4 two tokens that round alike, the larger one first / last; 5 several a few ulps apart;
    6, 7 negative values only, penalised."""
    nrows = 8

    def __init__(self, vocab, dtype, history=True, bias=True):
        g = torch.Generator().manual_seed(vocab)
        self.vocab, self.dtype = vocab, TYPES[dtype]
        x = torch.randn(8, vocab, generator=g).clamp_(-3, 3)
        b = torch.zeros(8, vocab)
        h = torch.full((8, 3), -1, dtype=torch.int64)
        lo, hi = 1, vocab - 2
        x[0, hi], x[1, hi] = 7.3, 13.7
        h[0, 1] = h[1, 0] = hi
        x[2, lo], b[2, lo] = 9.0, 0.1234567
        for r, (first, last) in ((3, (2.0 ** -25, 2.0 ** -26)), (4, (2.0 ** -26, 2.0 ** -25))):
            x[r, lo] = x[r, hi] = 5.0
            b[r, lo], b[r, hi] = first, last
        for i in range(min(4, vocab - 2)):
            x[5, 1 + i], b[5, 1 + i] = 8.0, 1.0 + 1e-7 * i
        h[5, 2] = 1
        x[6] = -9.0 - x[6].abs()
        x[7] = -5.0
        h[6] = h[7] = torch.tensor([0, 2, 2])
        b[6:] = torch.randn(2, vocab, generator=g) * 1e-3
        self.x = x.to(self.dtype)
        self.b = b if bias else None
        self.h = h if history else None
        self.rho, self.freq, self.pres = 1.3, 0.03, 0.01
        self.u = torch.tensor([0.5, 0.999, 0.0, 0.4, 0.6, 0.7, 0.3, 0.9])
        self.g = torch.tensor([1.0, -2.0, 0.5, 1.0, -1.0, 3.0, 0.25, 1.0])
        self.tokens = torch.tensor([hi, hi, lo, lo, hi, 2, 0, hi])

    def rounded(self):
        return True

    def rules(self, dev, bias=None):
        from dvae_amd.rules import TokenRules
        return TokenRules(self.rho, self.freq, self.pres, bias if bias is not None else None if self.b is None else self.b.to(dev))

    def history(self, dev):
        return None if self.h is None else self.h.to(dev)

    def row(self, r):
        c = R.counts(None if self.h is None else self.h[r].tolist(), 3, self.vocab)
        return R.ruled_row(self.x[r].double().numpy(), c, self.rho, self.freq, self.pres, None if self.b is None else self.b[r].numpy())

    def steps(self, y):
        """E: how far the kernel's value may be from the oracle's."""
        return 6 * 2.0 ** -52 * (np.abs(y).max() + 20.0)

    def doubles(self, y, temp):
        """Whether the row is computed in doubles whatever its vocabulary (away from the rule's borders)."""
        top = abs(y.max()) / temp
        return self.vocab <= 128 or top > 1000


def tolerance(case, y, lp, temp, drawn):
    tol = 4 * case.steps(y) / temp + U * abs(lp) + 1e-11
    return tol if drawn or case.doubles(y, temp) else tol + log_z_tol(case, y, temp)


VOCABS = [6, 128, 200, 500, 9000]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("temp", COLD)
@pytest.mark.parametrize("vocab", VOCABS)
def test_decisions_and_their_log_probability(cuda, vocab, temp, dtype):
    from dvae_amd.rules import choose
    case = Cold(vocab, dtype)
    for u in (None, case.u):
        got = choose(case.x.to(cuda), case.rules(cuda), case.history(cuda), temperature=temp, uniforms=None if u is None else u.to(cuda))
        for r in range(case.nrows):
            y, _ = case.row(r)
            t, lp = R.choose_row(y, temp, None if u is None else float(u[r]))
            assert int(got.tokens[r]) == t, (r, int(got.tokens[r]), t)
            same_or_close(float(got.logprob[r]), lp, tolerance(case, y, lp, temp, u is not None), "row %d" % r)


def check_gradients(cuda, case, temp, bias_kind):
    from dvae_amd.rules import token_logprob
    x = case.x.to(cuda).requires_grad_(True)
    b = case.b.to(cuda).requires_grad_(True) if case.b is not None else None
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda, b), case.history(cuda), temperature=temp)
    grads = torch.autograd.grad(lp, [x] + ([] if b is None else [b]), case.g.to(cuda))
    total, most, off = np.zeros(case.vocab), np.zeros(case.vocab), np.zeros(case.vocab)
    for r in range(case.nrows):
        y, slope = case.row(r)
        want, d, dv = R.logprob_row(y, slope, int(case.tokens[r]), temp, float(case.g[r]))
        same_or_close(lp[r].item(), np.float32(want) if abs(want) > 3.4e38 else want, tolerance(case, y, want, temp, False), "log p of row %d" % r)
        p = np.exp(R.log_softmax(y, temp)[0])
        scale = abs(float(case.g[r])) / temp
        err = scale * p * (4 * case.steps(y) / temp + 1e-11) + U * np.abs(dv) + 2.0 ** -150
        if not case.doubles(y, temp):
            err = err + scale * (U * LN2_3 + p * (U * np.abs(y) / temp + 4 * U + log_z_tol(case, y, temp))) + 3 * U * np.abs(dv)
        same_or_close(grads[0][r].double().cpu().numpy(), d, err * slope + (half(case.dtype) + 2 * U) * np.abs(d) + TINY[case.dtype],
                      "d logits of row %d" % r)
        total, most, off = total + dv, most + np.abs(dv), off + err
        if bias_kind == "rows":
            same_or_close(grads[1][r].double().cpu().numpy(), dv, err, "d bias of row %d" % r)
    if bias_kind == "shared":
        # an addition of the running sum rounds by at most U times the sum so far, and that is at most the sum of all |dv| (rows of
        # either sign: |total| may be far smaller)
        same_or_close(grads[1].double().cpu().numpy(), total, off + case.nrows * U * (most + off), "d bias")


LN2_3 = 3 * math.log(2.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("temp", COLD)
@pytest.mark.parametrize("vocab", VOCABS)
def test_log_probability_and_gradients(cuda, vocab, temp, dtype):
    check_gradients(cuda, Cold(vocab, dtype), temp, "rows")


@pytest.mark.parametrize("temp", [1e-4, 1e-9, 1e-37])
@pytest.mark.parametrize("vocab", VOCABS)
def test_gradients_without_a_bias(cuda, vocab, temp):
    check_gradients(cuda, Cold(vocab, "fp32", bias=False), temp, None)


class Shared(Cold):
    """The same rows under one bias, which is not exact beside any logit of the top."""

    def __init__(self, vocab, dtype, history):
        super().__init__(vocab, dtype, history)
        g = torch.Generator().manual_seed(7)
        self.b = torch.randn(vocab, generator=g) * 1e-3

    def row(self, r):
        c = R.counts(None if self.h is None else self.h[r].tolist(), 3, self.vocab)
        return R.ruled_row(self.x[r].double().numpy(), c, self.rho, self.freq, self.pres, self.b.numpy())


@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("temp", [1e-4, 1e-9, 1e-30])
@pytest.mark.parametrize("vocab", VOCABS)
def test_gradients_of_a_shared_bias(cuda, vocab, temp, dtype, history):
    check_gradients(cuda, Shared(vocab, dtype, history), temp, "shared")


@pytest.mark.parametrize("vocab", [200, 500, 9000])
def test_many_cold_rows(cuda, vocab):
    """Rows of one segment each (a wave decides them) and rows of several: 600 copies of the eight, every copy alike."""
    from dvae_amd.rules import choose, token_logprob
    case = Cold(vocab, "fp32")
    n = 600
    x, b, h = (t.repeat(n, 1).to(cuda) for t in (case.x, case.b, case.h))
    from dvae_amd.rules import TokenRules
    rules = TokenRules(case.rho, case.freq, case.pres, b)
    few = choose(case.x.to(cuda), case.rules(cuda), case.history(cuda), temperature=1e-10, uniforms=case.u.to(cuda))
    many = choose(x, rules, h, temperature=1e-10, uniforms=case.u.repeat(n).to(cuda))
    assert torch.equal(many.tokens, few.tokens.repeat(n))
    best = choose(x, rules, h, temperature=1e-10)
    lp = token_logprob(x, case.tokens.repeat(n).to(cuda), rules, h, temperature=1e-10)
    for r in range(8):
        y, _ = case.row(r)
        t, want = R.choose_row(y, 1e-10)
        assert (best.tokens[r::8] == t).all()
        tol = tolerance(case, y, want, 1e-10, True)
        assert (best.logprob[r::8] - want).abs().max() <= tol
        want = R.log_softmax(y, 1e-10)[0][int(case.tokens[r])]
        assert ((lp[r::8] - want).abs() <= tolerance(case, y, want, 1e-10, True)).all()


@pytest.mark.parametrize("temp", [0.02, 0.05, 0.2])
@pytest.mark.parametrize("vocab", [8, 200, 500, 9000])
@pytest.mark.parametrize("rows", [1, 600])
def test_a_token_that_is_nearly_everything(cuda, vocab, temp, rows):
    """Its log p is that of what the others leave, however its value rounds: rows 0 .. 2 of Cold, whose top stands 2.5 and more
    above values of at most 3 (T 0.02 .. 0.2: the others' share S is at most V e^-12.5).  Its weight is 1 exactly; the fp32 sum of 1 and S is
    rounded at most 8 + 6 times near 1 (a vector of 8 in the lane it is in, 6 steps of the wave), S itself is off by 2^-17 S (a
    thousandth of the bound on the weights of test_gpu_rules.py would do); doubles: 1e-11."""
    from dvae_amd.rules import TokenRules, choose, token_logprob
    case = Cold(vocab, "fp32")
    x, b, h = (t[:3].repeat(rows, 1).to(cuda) for t in (case.x, case.b, case.h))
    tokens = case.tokens[:3].repeat(rows).to(cuda)
    rules = TokenRules(case.rho, case.freq, case.pres, b)
    best = choose(x, rules, h, temperature=temp)
    assert torch.equal(best.tokens, tokens)
    lp = token_logprob(x, tokens, rules, h, temperature=temp)
    for r in range(3):
        y, _ = case.row(r)
        want = R.log_softmax(y, temp)[0][int(case.tokens[r])]
        assert want > -0.04
        tol = U * abs(want) + (14 * U + 2.0 ** -17 * abs(want) if vocab > 128 else 1e-11)
        for got in (best.logprob[r::3], lp[r::3]):
            assert (got.double() - want).abs().max() <= tol, (r, float(got[0]), want, tol)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [5, 100, 300, 9000])
def test_infinities_that_the_history_holds(cuda, vocab, dtype):
    """+-inf / 1.3 and +-inf * 1.3 are infinite, not NaN; in the other tokens nothing of them shows."""
    from dvae_amd.rules import TokenRules, apply_rules, choose
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(3, vocab, generator=g).to(TYPES[dtype])
    x[0, 1] = x[1, vocab - 1] = math.inf
    x[1, 0] = x[2, 2] = -math.inf
    h = torch.tensor([1, 0, vocab - 1, 2, 2])
    b = torch.randn(vocab, generator=g)
    for bias in (None, b):
        r = TokenRules(1.3, 0.25, 0.5, None if bias is None else bias.to(cuda))
        got = apply_rules(x.to(cuda), r, h.to(cuda)).double().cpu().numpy()
        for i in range(3):
            y, _ = R.ruled_row(x[i].double().numpy(), R.counts(h.tolist(), 5, vocab), 1.3, 0.25, 0.5, None if bias is None else bias.numpy())
            same_or_close(got[i], y, (half(TYPES[dtype]) + U) * np.abs(np.where(np.isfinite(y), y, 0.0)) + TINY[TYPES[dtype]], "row %d" % i)
        for u in (None, torch.full((3,), 0.5, device=cuda)):
            picked = choose(x.to(cuda), r, h.to(cuda), uniforms=u)
            assert picked.tokens[:2].tolist() == [-1, -1] and torch.isnan(picked.logprob[:2]).all() and int(picked.tokens[2]) >= 0


def test_a_repetition_penalty_near_zero(cuda):
    """x / 1e-310 is beyond every type: +inf, not NaN; 0 stays 0 and a negative value goes to 0."""
    from dvae_amd.rules import TokenRules, apply_rules
    for vocab in (5, 300):
        x = torch.zeros(2, vocab, device=cuda)
        x[:, 0], x[:, 1] = 2.0, -3.0
        got = apply_rules(x, TokenRules(1e-310), torch.tensor([0, 1, 2], device=cuda))
        assert torch.isinf(got[:, 0]).all() and (got[:, 0] > 0).all() and (got[:, 1:] == 0).all()


@pytest.mark.parametrize("vocab", [6, 200, 700, 9000])
def test_the_smallest_uniform_number_before_improbable_tokens(cuda, vocab):
    """u = 0 draws the first token that counts as probable -- here 2^-1010 of the largest is none, 2^-980 is one --, u = 1 the
    last one: never no token at all."""
    from dvae_amd.rules import choose
    for low, first in ((-200.0, vocab - 1), (-179.0, 0)):
        x = torch.full((2, vocab), low, device=cuda)
        x[0, vocab - 1] = 500.0
        x[1, 0] = 500.0
        got = choose(x, uniforms=torch.tensor([0.0, 1.0], device=cuda))
        assert got.tokens.tolist() == [first, 0 if first else vocab - 1]
        assert torch.isfinite(got.logprob).all()


@pytest.mark.parametrize("vocab", [6, 200, 700, 9000])
def test_values_beyond_fp32(cuda, vocab):
    """The lowest number times a penalty of 1.3 is -inf in fp32: log p -inf and no gradient from it, a row of nothing else is one
    whose rules leave nothing -- in every kernel."""
    from dvae_amd.rules import TokenRules, choose, token_logprob
    low = torch.finfo(torch.float32).min
    x = torch.zeros(3, vocab, device=cuda)
    x[:, 1] = low
    x[1, :] = low
    h = torch.tensor([[1] * vocab, list(range(vocab)), [1] * vocab], device=cuda)
    r = TokenRules(1.3)
    for u in (None, torch.full((3,), 0.5, device=cuda)):
        got = choose(x, r, h, uniforms=u)
        assert got.tokens.tolist()[1] == -1 and float(got.logprob[1]) == -math.inf
        assert got.tokens.tolist()[0] == got.tokens.tolist()[2] >= 0
    x.requires_grad_(True)
    lp = token_logprob(x, torch.tensor([1, 1, 0], device=cuda), r, h)
    dx, = torch.autograd.grad(lp, x, torch.ones(3, device=cuda))
    assert lp.tolist()[:2] == [-math.inf, -math.inf] and abs(float(lp[2]) + math.log(vocab - 1)) <= 1e-5
    assert torch.isfinite(dx).all() and (dx[1] == 0).all() and float(dx[2, 1]) == 0.0 and float(dx[0, 0]) < 0.0


class Far(Shared):
    """Logits near -1000 at T = 1: no ordinary maximum (2^-1443), and every token counts."""

    def __init__(self, vocab, dtype):
        super().__init__(vocab, dtype, True)
        g = torch.Generator().manual_seed(vocab + 1)
        self.x = (torch.randn(8, vocab, generator=g) * 2 - 1000.0).to(self.dtype)
        self.rho = 1.001
        self.h = torch.randint(0, vocab, (8, 3), generator=g)
        self.tokens = torch.randint(0, vocab, (8,), generator=g)

    def steps(self, y):
        return 6 * 2.0 ** -52 * 1100.0

    def doubles(self, y, temp):
        return True


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [6, 200, 500, 9000])
def test_rows_far_below_zero_under_a_bias(cuda, vocab, dtype):
    from dvae_amd.rules import choose
    case = Far(vocab, dtype)
    for u in (None, case.u):
        got = choose(case.x.to(cuda), case.rules(cuda), case.history(cuda), temperature=1.0, uniforms=None if u is None else u.to(cuda))
        for r in range(case.nrows):
            y, _ = case.row(r)
            t, lp = R.choose_row(y, 1.0, None if u is None else float(u[r]))
            assert int(got.tokens[r]) == t
            same_or_close(float(got.logprob[r]), lp, tolerance(case, y, lp, 1.0, True), "row %d" % r)
    check_gradients(cuda, case, 1.0, "shared")


@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("vocab", [200, 500, 9000])
def test_a_nan_gradient_in_a_cold_row(cuda, vocab, per_row):
    """It shows in every allowed place of its row and of the bias, an ignored or forbidden place stays 0; other rows are as they were."""
    from dvae_amd.rules import Grammar, TokenRules, token_logprob
    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(0)).to(cuda).requires_grad_()
    b = torch.full((4, vocab) if per_row else (vocab,), 0.1, device=cuda, requires_grad=True)
    allowed = torch.ones(1, vocab, dtype=torch.bool, device=cuda)
    allowed[0, ::7] = False
    t = torch.tensor([1, 2, -1, 3], device=cuda)
    lp = token_logprob(x, t, TokenRules(bias=b, grammar=Grammar(allowed)), state=torch.zeros(4, dtype=torch.int32, device=cuda),
                       temperature=1e-5)
    dx, db = torch.autograd.grad(lp, [x, b], torch.tensor([1.0, math.nan, math.nan, 0.0], device=cuda))
    assert torch.isnan(dx[1][allowed[0]]).all() and (dx[1][~allowed[0]] == 0).all()
    assert torch.isfinite(dx[0]).all() and (dx[2:] == 0).all()
    row = db[1] if per_row else db
    assert torch.isnan(row[allowed[0]]).all() and (row[~allowed[0]] == 0).all()
    if per_row:
        assert torch.equal(db[[0, 2, 3]], dx[[0, 2, 3]])
