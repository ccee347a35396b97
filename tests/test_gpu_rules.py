"""GPU: token rules -- values, tokens, log-probabilities and gradients -- against oracle/rules_ref.py (64 bits, row by row).

Tolerances.  u = 2^-24 is half a step of fp32, h half a step of the result's type.
* values: one rounding to fp32 of the exact value, one to the type: (h + u) |x4|, and half a step of the smallest number.
* log p of a draw: doubles, rounded once: u |lp| + 1e-11.  From fp32 sums (greedy, token_logprob) also log Z's error: a
  weight 2^a, a = (x4 - ref) k, is off by the roundings of x4 (u |x4| k, if there is a bias or a history), of the
  difference, of k and of their product (3 u |a|), of exp2 (2 u, one step) -- times ln 2 where it is an exponent.  The sum
  over all weights of p |a| is at most 8 (the reference may be 2^8 low) + log2 V.  Sums: 64 steps of a lane and a
  vector of 8, 6 of the wave, in the worst case one rounding each.  The lane's and the segment's rescaling: another 3 |a| + 2 each.
  Together  LZ = u (ln2 (3 (24 + 3 log2 V) + max|x4| k) + 6 + 80).
* gradients: d = g / T ([v = t] - p), p off by p (u ln2 (3 |a| + |x4| k) + 2 u + LZ + 2 u) with p |a| <= 1 (2^-|a| |a| < 1),
  then three roundings of d and the one to the type.
* the bias gradient: its rows' errors, plus one rounding of the running sum per row.
"""
import math

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from oracle import rules_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LN2 = math.log(2.0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


class Case:
    """Inputs of one call on the CPU, made from a seed; rows() gives the oracle's view of each row."""

    def __init__(self, rows, vocab, dtype="fp32", L=0, ragged=False, index=torch.int64, per_row=False, bias=None, states=0,
                 free=False, share=0.6, seed=0, pad=0, scale=3.0, drawn=False, junk=False):
        g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + vocab)
        self.dtype = TYPES[dtype]
        self.big = (torch.randn(rows, vocab + pad, generator=g) * scale).to(self.dtype)
        self.history = self.lengths = self.state = None
        if L:
            h = (torch.rand(rows, L, generator=g) ** 2 * vocab).long().clamp_(max=vocab - 1)
            if junk:
                wrong = torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (rows, L), generator=g)]
                h = torch.where(torch.rand(rows, L, generator=g) < 0.3, wrong, h)
            self.history = h.to(index)
            if ragged:
                self.lengths = torch.randint(0, L + 1, (rows,), generator=g, dtype=torch.int32)
                self.lengths[0] = 0
        if per_row:
            self.rho, self.freq = 0.7 + torch.rand(rows, generator=g), torch.rand(rows, generator=g) - 0.3
            self.pres, self.temp = torch.rand(rows, generator=g), 0.3 + torch.rand(rows, generator=g)
        else:
            self.rho, self.freq, self.pres, self.temp = 1.1, 0.3, 0.2, 0.7
        self.bias = {None: None, "shared": torch.randn(vocab, generator=g),
                     "rows": torch.randn(rows, vocab, generator=g)}[bias]
        self.allowed = self.next = None
        if states:
            self.allowed = torch.rand(states, vocab, generator=g) < share
            if states > 1:
                self.allowed[1] = False                       # a state that leaves nothing
            self.next = torch.randint(-1, states + 1, (states, vocab), generator=g, dtype=torch.int32)
            self.state = torch.randint(-1 if free else 0, states + (1 if free else 0), (rows,), generator=g, dtype=torch.int32)
        self.u = torch.rand(rows, generator=g) if drawn else None
        if drawn and rows > 2:
            self.u[0], self.u[1] = 0.0, 1.0 - 2.0 ** -24
        self.tokens = torch.randint(0, vocab, (rows,), generator=g)
        self.g = torch.randn(rows, generator=g)
        self.nrows, self.vocab = rows, vocab

    @property
    def logits(self):
        return self.big[:, :self.vocab]

    def rules(self, dev, bias=None):
        from dvae_amd.rules import Grammar, TokenRules
        d = [v.to(dev) if torch.is_tensor(v) else v for v in (self.rho, self.freq, self.pres)]
        b = bias if bias is not None else None if self.bias is None else self.bias.to(dev)
        gr = None if self.allowed is None else Grammar(self.allowed.to(dev), self.next.to(dev))
        return TokenRules(d[0], d[1], d[2], b, gr)

    def kw(self, dev):
        def to(t):
            return None if t is None else t.to(dev)
        return dict(history=to(self.history), lengths=to(self.lengths), state=to(self.state))

    def temperature(self, dev):
        return self.temp.to(dev) if torch.is_tensor(self.temp) else self.temp

    def row(self, r):
        """-> (x4, slope, allowed or None, temperature) of a row, float64."""
        def at(v):
            return float(v[r]) if torch.is_tensor(v) else v
        L = 0 if self.history is None else self.history.shape[1]
        n = L if self.lengths is None else int(self.lengths[r])
        c = R.counts(None if self.history is None else self.history[r].tolist(), n, self.vocab)
        b = None if self.bias is None else (self.bias if self.bias.dim() == 1 else self.bias[r]).numpy()
        al = None
        if self.allowed is not None and 0 <= int(self.state[r]) < self.allowed.shape[0]:
            al = self.allowed[int(self.state[r])].numpy()
        y, slope = R.ruled_row(self.logits[r].double().numpy(), c, at(self.rho), at(self.freq), at(self.pres), b, al)
        return y, slope, al, at(self.temp)

    def rounded(self):
        return self.bias is not None or self.history is not None


def half(dtype):
    return torch.finfo(dtype).eps / 2


def log_z_tol(case, y, temp):
    fin = y[np.isfinite(y)]
    top = np.abs(fin).max() if len(fin) else 0.0
    k = 1.0 / (LN2 * temp)
    return U * (LN2 * (3 * (24 + 3 * math.log2(max(case.vocab, 2))) + (top * k if case.rounded() else 0.0)) + 86)


def same_or_close(got, want, tol, what):
    got, want, tol = (np.asarray(v, dtype=np.float64) for v in (got, want, tol))
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what + ": infinities in other places"
    with np.errstate(invalid="ignore"):
        err = np.abs(got - want)
    bad = ~odd & ~(err <= np.broadcast_to(tol, err.shape))
    assert not bad.any(), "%s: %d of %d off, worst %.3e where %.3e is allowed" % (
        what, bad.sum(), bad.size, err[bad].max(), np.broadcast_to(tol, err.shape)[bad][err[bad].argmax()])


SHAPES = [
    dict(rows=1, vocab=1), dict(rows=3, vocab=2, L=3, dtype="bf16"), dict(rows=5, vocab=7, L=9, states=3, bias="shared"),
    dict(rows=70, vocab=8, L=7, ragged=True, states=4, free=True, dtype="fp32", index=torch.int32, per_row=True),
    dict(rows=9, vocab=31, dtype="fp16", states=3), dict(rows=4, vocab=33, dtype="bf16", L=5, pad=3, bias="rows"),
    dict(rows=6, vocab=63, L=200, ragged=True, junk=True), dict(rows=6, vocab=64, states=2, dtype="bf16", bias="shared"),
    dict(rows=6, vocab=65, L=20, ragged=True, dtype="fp16", pad=1), dict(rows=7, vocab=255, per_row=True, L=40, pad=2),
    dict(rows=5, vocab=256, bias="shared"), dict(rows=5, vocab=257, dtype="bf16", L=300, junk=True, index=torch.int32),
    dict(rows=3, vocab=511, dtype="fp16", bias="rows", states=5), dict(rows=3, vocab=513, dtype="bf16", L=64, states=2, free=True),
    dict(rows=2, vocab=1025, L=1000, ragged=True), dict(rows=5, vocab=2049, dtype="fp16", L=33, per_row=True, bias="shared"),
    dict(rows=3, vocab=4095, dtype="bf16", L=12, pad=7), dict(rows=2, vocab=4096, states=3), dict(rows=2, vocab=4097, L=100, dtype="bf16"),
    dict(rows=3, vocab=8193, dtype="fp16", bias="shared", states=4, L=50, ragged=True, pad=5),
    dict(rows=1, vocab=16384, L=5000, dtype="bf16"), dict(rows=2, vocab=16385, per_row=True, L=10, bias="rows"),
    dict(rows=2, vocab=50021, dtype="bf16", L=999, ragged=True, bias="shared", states=3, per_row=True, index=torch.int32),
    dict(rows=1, vocab=70001, L=70000, dtype="fp32"), dict(rows=2, vocab=300, L=66000, ragged=True, index=torch.int32, dtype="bf16"),
]


def ident(c):
    return "-".join("%s%s" % (k, str(v).replace("torch.", "")) for k, v in c.items())


@pytest.mark.parametrize("shape", SHAPES, ids=ident)
def test_apply(cuda, shape):
    from dvae_amd.rules import apply_rules
    case = Case(seed=1, **shape)
    x = case.big.to(cuda)[:, :case.vocab]
    got = apply_rules(x, case.rules(cuda), **case.kw(cuda))
    assert got.dtype == case.dtype and got.shape == x.shape
    assert torch.equal(x.cpu(), case.logits)                     # the logits stay
    for r in range(case.nrows):
        y, _, _, _ = case.row(r)
        tol = (half(case.dtype) + U) * np.abs(np.where(np.isfinite(y), y, 0.0)) + TINY[case.dtype]
        same_or_close(got[r].double().cpu().numpy(), y, tol, "row %d" % r)
    # in place, the same bits, and what lies between the rows is left alone
    big = case.big.to(cuda)
    z = big[:, :case.vocab]
    assert apply_rules(z, case.rules(cuda), out=z, **case.kw(cuda)) is z
    assert torch.equal(z, got) and torch.equal(big[:, case.vocab:].cpu(), case.big[:, case.vocab:])


@pytest.mark.parametrize("drawn", [False, True], ids=["greedy", "drawn"])
@pytest.mark.parametrize("shape", SHAPES, ids=ident)
def test_choose(cuda, shape, drawn):
    from dvae_amd.rules import choose
    case = Case(seed=2, drawn=drawn, **shape)
    x = case.big.to(cuda)[:, :case.vocab]
    got = choose(x, case.rules(cuda), temperature=case.temperature(cuda), uniforms=case.u.to(cuda) if drawn else None,
                 **case.kw(cuda))
    assert got.tokens.dtype == torch.int64 and got.logprob.dtype == torch.float32
    tokens = got.tokens.tolist()
    for r in range(case.nrows):
        y, _, _, temp = case.row(r)
        t, lp = R.choose_row(y, temp, float(case.u[r]) if drawn else None)
        assert tokens[r] == t, (r, tokens[r], t)
        tol = U * abs(lp) + 1e-11 + (0.0 if drawn else log_z_tol(case, y, temp)) if math.isfinite(lp) else 0.0
        same_or_close(float(got.logprob[r]), lp, tol, "row %d" % r)
        if case.state is not None:
            s = int(case.state[r])
            want = int(case.next[s, t]) if t >= 0 and 0 <= s < case.next.shape[0] else s
            assert int(got.state[r]) == want
    if case.state is None:
        assert got.state is None


def check_logprob(cuda, case, x, bias, lp, dx, db, g, some=None):
    want_db = np.zeros((case.nrows, case.vocab))
    tol_db = np.zeros((case.nrows, case.vocab))
    for r in range(case.nrows) if some is None else some:
        y, slope, al, temp = case.row(r)
        want, d, dv = R.logprob_row(y, slope, int(case.tokens[r]), temp, float(g[r]), al)
        lz = log_z_tol(case, y, temp)
        same_or_close(lp[r].item(), want, (U * abs(want) + lz) if math.isfinite(want) else 0.0, "log p of row %d" % r)
        p = np.exp(R.log_softmax(y, temp)[0])
        scale = abs(float(g[r])) / temp
        fin = np.where(np.isfinite(y), np.abs(y), 0.0)
        err = scale * (U * LN2 * 3 + p * ((U * LN2 * fin / (LN2 * temp) if case.rounded() else 0.0) + 4 * U + lz)) + 4 * U * np.abs(dv)
        want_db[r], tol_db[r] = dv, err
        tol = err * slope + (half(case.dtype) + U) * np.abs(d) + TINY[case.dtype]
        same_or_close(dx[r].double().cpu().numpy(), d, tol, "d logits of row %d" % r)
    if db is not None and db.dim() == 2:
        same_or_close(db.double().cpu().numpy(), want_db, tol_db, "d bias")
    elif db is not None:
        total = np.abs(want_db).sum(0)
        same_or_close(db.double().cpu().numpy(), want_db.sum(0), tol_db.sum(0) + case.nrows * U * (total + tol_db.sum(0)), "d bias")


@pytest.mark.parametrize("shape", SHAPES, ids=ident)
def test_logprob_and_gradients(cuda, shape):
    from dvae_amd.rules import token_logprob
    case = Case(seed=3, **shape)
    if case.nrows > 2:
        case.tokens[2] = -100                                    # an ignored row
    x = case.big.to(cuda)[:, :case.vocab].requires_grad_(True)
    b = None if case.bias is None else case.bias.to(cuda).requires_grad_(True)
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda, b), temperature=case.temperature(cuda), **case.kw(cuda))
    grads = torch.autograd.grad(lp, [x] + ([] if b is None else [b]), case.g.to(cuda))
    assert lp.dtype == torch.float32 and grads[0].dtype == case.dtype and grads[0].shape == x.shape
    check_logprob(cuda, case, x, b, lp, grads[0], None if b is None else grads[1], case.g)
    # the same bits again, and without the bias's gradient
    lp2 = token_logprob(x, case.tokens.to(cuda), case.rules(cuda, b), temperature=case.temperature(cuda), **case.kw(cuda))
    again = torch.autograd.grad(lp2, [x] + ([] if b is None else [b]), case.g.to(cuda))
    assert torch.equal(lp.nan_to_num(7.0), lp2.nan_to_num(7.0)) and all(torch.equal(a, c) for a, c in zip(grads, again))


def test_many_rows_share_one_bias(cuda):
    from dvae_amd.rules import token_logprob
    case = Case(rows=700, vocab=37, dtype="fp32", L=6, ragged=True, bias="shared", states=4, per_row=True, seed=9)
    x, b = case.logits.to(cuda).requires_grad_(True), case.bias.to(cuda).requires_grad_(True)
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda, b), temperature=case.temperature(cuda), **case.kw(cuda))
    dx, db = torch.autograd.grad(lp, [x, b], case.g.to(cuda))
    check_logprob(cuda, case, x, b, lp, dx, db, case.g)


@pytest.mark.parametrize("shape", [dict(vocab=8, L=7, index=torch.int32, states=5, free=True),
                                   dict(vocab=5, L=200, ragged=True, dtype="bf16", bias="shared", per_row=True, junk=True),
                                   dict(vocab=16, L=9, dtype="fp16", bias="rows", states=3, per_row=True, pad=1),
                                   dict(vocab=11, L=3, states=4), dict(vocab=1), dict(vocab=8, L=255),
                                   dict(vocab=100, L=32, dtype="bf16", states=3, per_row=True),
                                   dict(vocab=128, dtype="fp16", bias="rows"), dict(vocab=33, L=40, pad=2)], ids=ident)
def test_many_rows_of_a_few_tokens(cuda, shape):
    """32800 rows, histories short enough for groups of lanes, which compute in doubles.  The oracle sees 200 rows spread over them (the bias gradient: all)."""
    from dvae_amd.rules import apply_rules, choose, token_logprob
    rows = 32800
    case = Case(rows=rows, seed=12, drawn=True, **shape)
    x, kw, temp = case.big.to(cuda)[:, :case.vocab], case.kw(cuda), case.temperature(cuda)
    some = list(range(0, rows, 167)) + [rows - 1]
    got = apply_rules(x, case.rules(cuda), **kw).double().cpu().numpy()
    draw = choose(x, case.rules(cuda), temperature=temp, uniforms=case.u.to(cuda), **kw)
    best = choose(x, case.rules(cuda), temperature=temp, **kw)
    picked = [(c.tokens.tolist(), c.logprob.tolist(), None if c.state is None else c.state.tolist()) for c in (draw, best)]
    x = x.requires_grad_(True)
    shared = case.bias is not None and case.bias.dim() == 1
    b = case.bias.to(cuda).requires_grad_(True) if case.bias is not None else None
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda, b), temperature=temp, **kw)
    grads = torch.autograd.grad(lp, [x] + ([] if b is None else [b]), case.g.to(cuda))
    dx, values = grads[0].double().cpu().numpy(), lp.tolist()
    total, off = np.zeros(case.vocab), np.zeros(case.vocab)
    for r in (range(rows) if shared else some):
        y, slope, al, t = case.row(r)
        want, d, dv = R.logprob_row(y, slope, int(case.tokens[r]), t, float(case.g[r]), al)
        same_or_close(values[r], want, U * abs(want) + 1e-11 if math.isfinite(want) else 0.0, "log p of row %d" % r)
        # doubles but for 1 / Z and the maximum, each rounded once: 2 roundings of p, one of d and the type's
        p = np.exp(R.log_softmax(y, t)[0])
        scale = abs(float(case.g[r])) / t
        fin = np.where(np.isfinite(y), np.abs(y), 0.0).max()
        err = scale * p * (2 * U + U * fin / t) + U * np.abs(dv)
        same_or_close(dx[r], d, err * slope + (half(case.dtype) + U) * np.abs(d) + TINY[case.dtype], "d logits of row %d" % r)
        total, off = total + dv, off + err + rows * U * np.abs(dv)
        if r in (some if not shared else some[:50]):
            same_or_close(got[r], y, (half(case.dtype) + U) * np.abs(np.where(np.isfinite(y), y, 0)) + TINY[case.dtype], "row %d" % r)
            for (tok, lps, st), u in zip(picked, (float(case.u[r]), None)):
                k, l = R.choose_row(y, t, u)
                assert tok[r] == k, (r, tok[r], k)
                same_or_close(lps[r], l, U * abs(l) + 1e-11 if math.isfinite(l) else 0.0, "row %d" % r)
                if st is not None:
                    s = int(case.state[r])
                    assert st[r] == (int(case.next[s, k]) if k >= 0 and 0 <= s < case.next.shape[0] else s)
    if shared:
        same_or_close(grads[1].double().cpu().numpy(), total, off, "d bias")
    elif b is not None:
        assert grads[1].shape == b.shape


@pytest.mark.parametrize("shape", [dict(vocab=700, L=40, ragged=True, states=4, free=True, per_row=True),
                                   dict(vocab=1900, dtype="bf16", L=9, bias="rows", index=torch.int32, pad=3),
                                   dict(vocab=2048, dtype="fp16", states=3), dict(vocab=1025, L=600, junk=True),
                                   dict(vocab=13, L=256, states=2), dict(vocab=90, L=33, dtype="bf16")], ids=ident)
def test_many_rows_of_a_middle_vocabulary(cuda, shape):
    """4200 rows, more tokens or history than groups of lanes take: a wave a row, fp32 sums.  The oracle sees 60 of them."""
    from dvae_amd.rules import apply_rules, choose, token_logprob
    rows = 4200
    case = Case(rows=rows, seed=13, drawn=True, **shape)
    x, kw, temp = case.big.to(cuda)[:, :case.vocab], case.kw(cuda), case.temperature(cuda)
    got = apply_rules(x, case.rules(cuda), **kw)
    draw = choose(x, case.rules(cuda), temperature=temp, uniforms=case.u.to(cuda), **kw)
    best = choose(x, case.rules(cuda), temperature=temp, **kw)
    picked = [(c.tokens.tolist(), c.logprob.tolist(), None if c.state is None else c.state.tolist()) for c in (draw, best)]
    x = x.requires_grad_(True)
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda), temperature=temp, **kw)
    (dx,) = torch.autograd.grad(lp, x, case.g.to(cuda))
    some = list(range(0, rows, 71)) + [rows - 1]
    for r in some:
        y, _, _, t = case.row(r)
        same_or_close(got[r].double().cpu().numpy(), y,
                      (half(case.dtype) + U) * np.abs(np.where(np.isfinite(y), y, 0)) + TINY[case.dtype], "row %d" % r)
        for (tok, lps, st), u in zip(picked, (float(case.u[r]), None)):
            k, l = R.choose_row(y, t, u)
            assert tok[r] == k, (r, tok[r], k)
            tol = U * abs(l) + 1e-11 + (0.0 if u is not None else log_z_tol(case, y, t)) if math.isfinite(l) else 0.0
            same_or_close(lps[r], l, tol, "row %d" % r)
            if st is not None:
                s = int(case.state[r])
                assert st[r] == (int(case.next[s, k]) if k >= 0 and 0 <= s < case.next.shape[0] else s)
    check_logprob(cuda, case, x, None, lp, dx, None, case.g, some)


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's own log p along directions of +-1: the third derivative of a log-sum-exp along
    such a direction is a third central moment of a variable of +-1/T, at most 0.77 / T^3 (the Bernoulli extreme,
    max 8 q (1 - q)(1 - 2 q)): truncation h^2 / 6 of it; log p itself is off by 2 tolerances over 2 h."""
    from dvae_amd.rules import token_logprob
    case = Case(rows=6, vocab=19, L=5, bias="shared", states=0, seed=4)
    keep = case.big.abs() < 0.25
    case.big[keep] += 0.5 * torch.sign(case.big[keep] + 1e-3)     # away from the penalty's kink at 0
    x, b = case.logits.to(cuda).requires_grad_(True), case.bias.to(cuda).requires_grad_(True)
    tok, temp = case.tokens.to(cuda), case.temp
    lp = token_logprob(x, tok, case.rules(cuda, b), temperature=temp, **case.kw(cuda))
    dx, db = torch.autograd.grad(lp.sum(), [x, b])
    h = 2.0 ** -5
    lz = max(log_z_tol(case, case.row(r)[0], temp) for r in range(6)) + U * 30
    gen = torch.Generator().manual_seed(1)
    for what in ("logits", "bias"):
        for _ in range(3):
            v = torch.randint(0, 2, x.shape if what == "logits" else b.shape, generator=gen).to(cuda) * 2.0 - 1.0
            def f(s):
                xs = x.detach() + s * v if what == "logits" else x.detach()
                bs = b.detach() + s * v if what == "bias" else b.detach()
                return token_logprob(xs, tok, case.rules(cuda, bs), temperature=temp, **case.kw(cuda)).double()
            slope = ((f(h) - f(-h)) / (2 * h)).sum().item()
            want = ((dx * v).double().sum() if what == "logits" else (db * v).double().sum()).item()
            steps = 1.1 if what == "logits" else 1.0              # a counted logit moves by up to rho
            tol = 6 * (h * h / 6 * 0.77 * (2 * steps / temp) ** 3 + lz / h) + 6 * 40 * U
            assert abs(slope - want) <= tol, (what, slope, want, tol)


# ---- rows that are not ordinary ----
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [6, 300, 9000])
def test_masked_places_hold_anything(cuda, vocab, dtype):
    """NaN, infinities and the lowest number where the grammar forbids: nothing of it shows."""
    from dvae_amd.rules import apply_rules, choose, token_logprob
    case = Case(rows=8, vocab=vocab, dtype=dtype, states=3, L=4, bias="shared", seed=5)
    case.state = torch.tensor([0, 2] * 4, dtype=torch.int32)
    case.allowed[:, 0] = True
    off = ~case.allowed[case.state.long()]
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(case.dtype).min]).to(case.dtype)
    case.big = torch.where(off, junk[torch.arange(vocab) % 4], case.big)
    case.bias = torch.where(off.all(0), torch.tensor(math.nan), case.bias)
    case.tokens[:] = 0
    x = case.big.to(cuda)
    for r, row in enumerate(apply_rules(x, case.rules(cuda), **case.kw(cuda)).double().cpu().numpy()):
        y = case.row(r)[0]
        same_or_close(row, y, (half(case.dtype) + U) * np.abs(np.where(np.isfinite(y), y, 0)) + TINY[case.dtype], "row %d" % r)
    for u in (None, torch.rand(8, generator=torch.Generator().manual_seed(0))):
        got = choose(x, case.rules(cuda), temperature=0.7, uniforms=None if u is None else u.to(cuda), **case.kw(cuda))
        assert got.tokens.tolist() == [R.choose_row(case.row(r)[0], 0.7, None if u is None else float(u[r]))[0] for r in range(8)]
        assert torch.isfinite(got.logprob).all()
    x.requires_grad_(True)
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda), temperature=0.7, **case.kw(cuda))
    (dx,) = torch.autograd.grad(lp, x, case.g.to(cuda))
    check_logprob(cuda, case, x, None, lp, dx, None, case.g)
    assert (dx.cpu()[off] == 0).all()


@pytest.mark.parametrize("vocab", [5, 700, 9001])
def test_allowed_nan_and_infinity_show(cuda, vocab):
    from dvae_amd.rules import choose, token_logprob
    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(0))
    x[0, vocab - 1] = math.nan
    x[1, vocab // 2] = math.inf
    x[2, :] = -math.inf
    x[3, :vocab - 1] = -math.inf                                 # one token left
    x = x.to(cuda)
    for u in (None, torch.full((4,), 0.5, device=cuda)):
        got = choose(x, uniforms=u)
        assert got.tokens.tolist() == [-1, -1, -1, vocab - 1]
        lp = got.logprob.tolist()
        # the one token left has p = 1: log Z is that of 2^a 2^-a, each power off by at most 4e-14 of itself
        assert math.isnan(lp[0]) and math.isnan(lp[1]) and lp[2] == -math.inf and abs(lp[3]) <= 1e-13
    x.requires_grad_(True)
    lp = token_logprob(x, torch.zeros(4, dtype=torch.int64, device=cuda))
    (dx,) = torch.autograd.grad(lp.sum(), x)
    assert math.isnan(lp[0]) and math.isnan(lp[1]) and lp[2] == -math.inf and lp[3] == -math.inf
    assert torch.isnan(dx[0]).all() and (dx[2] == 0).all() and dx[3, vocab - 1] == -1.0 and dx[3, 0] == 1.0


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [9, 5000])
def test_rows_of_the_lowest_number(cuda, vocab, dtype):
    """Masks made of the type's lowest value instead of -inf: a row of nothing else is a uniform one."""
    from dvae_amd.rules import choose, token_logprob
    low = torch.finfo(TYPES[dtype]).min
    x = torch.full((2, vocab), low, dtype=TYPES[dtype], device=cuda)
    x[1, 3] = 0.25
    for temp in (0.5, 1.0):
        got = choose(x, temperature=temp, uniforms=torch.tensor([0.5, 0.5], device=cuda))
        assert got.tokens.tolist() == [vocab // 2 if vocab % 2 == 0 else vocab // 2, 3]
        assert abs(float(got.logprob[0]) + math.log(vocab)) <= U * 10 and abs(float(got.logprob[1])) <= 1e-13
        assert choose(x, temperature=temp).tokens.tolist() == [0, 3]
        lp = token_logprob(x, torch.tensor([vocab - 1, 3], device=cuda), temperature=temp)
        assert abs(float(lp[0]) + math.log(vocab)) <= 1e-5 and abs(float(lp[1])) <= 1e-5


def test_numbers_that_are_not_uniform_ones(cuda):
    """u below 0 is 0, u from 1 on the last token with a probability, NaN no token."""
    from dvae_amd.rules import choose
    for vocab in (6, 5000):
        x = torch.zeros(5, vocab, device=cuda)
        x[:, 0] = x[:, vocab - 1] = -math.inf
        u = torch.tensor([-1.0, 0.0, 1.0, 7.0, math.nan], device=cuda)
        got = choose(x, uniforms=u)
        assert got.tokens.tolist() == [1, 1, vocab - 2, vocab - 2, -1]
        assert math.isnan(float(got.logprob[4])) and torch.isfinite(got.logprob[:4]).all()


def test_temperatures_of_rows_that_are_no_temperatures(cuda):
    from dvae_amd.rules import choose, token_logprob
    for vocab in (6, 5000):
        x = torch.randn(5, vocab, device=cuda)
        t = torch.tensor([0.0, -1.0, math.inf, math.nan, 1.0], device=cuda)
        for u in (None, torch.rand(5, device=cuda)):
            got = choose(x, temperature=t, uniforms=u)
            assert got.tokens[:4].tolist() == [-1] * 4 and torch.isnan(got.logprob[:4]).all()
            assert int(got.tokens[4]) >= 0 and torch.isfinite(got.logprob[4])
        lp = token_logprob(x, torch.zeros(5, dtype=torch.int64, device=cuda), temperature=t)
        assert torch.isnan(lp[:4]).all() and torch.isfinite(lp[4])


def test_temperatures_at_the_ends(cuda):
    """1e37: every allowed token alike; 1e-37: only the largest has a probability (a tie: two halves)."""
    from dvae_amd.rules import Grammar, TokenRules, choose, token_logprob
    for vocab in (6, 500, 9000):
        x = torch.randn(3, vocab, generator=torch.Generator().manual_seed(0)).to(cuda)
        x[1] = torch.finfo(torch.float32).min
        x[2, :2] = 50.0
        allowed = torch.ones(1, vocab, dtype=torch.bool, device=cuda)
        allowed[0, vocab - 1] = False
        r, st = TokenRules(grammar=Grammar(allowed)), torch.zeros(3, dtype=torch.int32, device=cuda)
        flat = choose(x, r, state=st, temperature=1e37, uniforms=torch.full((3,), 0.999999, device=cuda))
        assert flat.tokens.tolist()[0] == vocab - 2 and flat.tokens.tolist()[2] == vocab - 2
        assert torch.allclose(flat.logprob[[0, 2]].double(), torch.full((2,), -math.log(vocab - 1), dtype=torch.float64, device=cuda),
                              rtol=2 * U, atol=0)
        cold = choose(x, r, state=st, temperature=1e-37, uniforms=torch.full((3,), 0.75, device=cuda))
        best = int(x[0, :vocab - 1].argmax())
        assert cold.tokens.tolist() == [best, (3 * (vocab - 1)) // 4, 1] and abs(float(cold.logprob[0])) <= 1e-13
        assert abs(float(cold.logprob[2]) + math.log(2)) <= 2 * U
        t = torch.tensor([best, 0, 1], device=cuda)
        lp = token_logprob(x, t, r, state=st, temperature=1e-37)
        assert abs(lp[0].item()) <= U and abs(lp[1].item() + math.log(vocab - 1)) <= 1e-5 and abs(lp[2].item() + math.log(2)) <= 2 * U


@pytest.mark.parametrize("shift", [4096.0, -4096.0])
def test_rows_far_from_zero(cuda, shift):
    """A softmax does not see a shift (exact here: multiples of 2^-6): exponents of +-12000 and more."""
    from dvae_amd.rules import choose, token_logprob
    for vocab in (7, 500, 9000):
        g = torch.Generator().manual_seed(3)
        x = (torch.randn(8, vocab, generator=g) * 3 * 64).round().div(64).to(cuda)
        u, tok = torch.rand(8, generator=g).to(cuda), torch.randint(0, vocab, (8,), generator=g).to(cuda)
        hist = torch.randint(0, vocab, (8, 5), generator=g).to(cuda)
        for kw in (dict(), dict(history=hist)):
            for uu in (u, None):
                a, b = choose(x, uniforms=uu, temperature=0.5, **kw), choose(x + shift, uniforms=uu, temperature=0.5, **kw)
                assert torch.equal(a.tokens, b.tokens)
                assert float((a.logprob - b.logprob).abs().max()) <= 4 * U * (float(a.logprob.abs().max()) + 100)
            a, b = token_logprob(x, tok, temperature=0.5, **kw), token_logprob(x + shift, tok, temperature=0.5, **kw)
            # both sums are of the same differences x4 - ref: they differ by the segments' joins only
            assert float((a - b).abs().max()) <= 4 * U * (float(a.abs().max()) + 100)


def test_ties_go_to_the_lowest_index(cuda):
    from dvae_amd.rules import TokenRules, choose
    for vocab in (8, 600, 20000):
        x = torch.zeros(3, vocab, device=cuda, dtype=torch.bfloat16)
        x[1, vocab - 1] = x[1, vocab // 2] = 2.0
        x[2, vocab - 1] = 5.0                                    # 5 / 1.25 ties with 4
        x[2, vocab - 2] = 4.0
        hist = torch.full((3, 1), vocab - 1, device=cuda)
        assert choose(x).tokens.tolist() == [0, vocab // 2, vocab - 1]
        assert choose(x, TokenRules(repetition=1.25), history=hist).tokens.tolist() == [0, vocab // 2, vocab - 2]


def test_values_that_round_alike_are_told_apart(cuda):
    """x + b of two tokens that fp32 rounds to one number: the larger exact one wins whatever its index."""
    from dvae_amd.rules import TokenRules, choose
    for vocab in (8, 700, 20000):
        x = torch.full((2, vocab), -9.0, device=cuda)
        bias = torch.zeros(2, vocab, device=cuda)
        lo, hi = 1, vocab - 2
        x[:, lo] = x[:, hi] = 1.0
        bias[0, lo], bias[0, hi] = 2.0 ** -30, 2.0 ** -29
        bias[1, lo], bias[1, hi] = 2.0 ** -29, 2.0 ** -30
        assert choose(x, TokenRules(bias=bias)).tokens.tolist() == [hi, lo]


def test_presence_inf_forbids_what_was_there(cuda):
    from dvae_amd.rules import TokenRules, choose
    for vocab in (5, 4000):
        x = torch.arange(vocab, dtype=torch.float32, device=cuda).flip(0).repeat(2, 1)
        hist = torch.tensor([[0, 1, 2], [0, 0, 7]], device=cuda)
        got = choose(x, TokenRules(presence=math.inf), history=hist)
        assert got.tokens.tolist() == [3, 1]
    every = torch.arange(5, device=cuda).repeat(1, 1)
    got = choose(torch.zeros(1, 5, device=cuda), TokenRules(presence=math.inf), history=every, uniforms=torch.zeros(1, device=cuda))
    assert got.tokens.tolist() == [-1] and float(got.logprob) == -math.inf


# ---- layouts ----
def test_leading_axes_and_shared_histories(cuda):
    from dvae_amd.rules import TokenRules, apply_rules, choose, token_logprob
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 4, 29, generator=g).to(cuda)
    hist = torch.randint(0, 29, (3, 6), generator=g).to(cuda)
    lens = torch.randint(0, 7, (3, 4), generator=g).to(cuda)
    r = TokenRules(1.3, 0.2, 0.1)
    flat = hist[:, None].expand(3, 4, 6).reshape(12, 6)
    want = apply_rules(x.view(12, 29), r, flat, lens.view(12))
    assert torch.equal(apply_rules(x, r, hist, lens).view(12, 29), want)
    assert torch.equal(choose(x, r, hist, lens).tokens.view(12), choose(x.view(12, 29), r, flat, lens.view(12)).tokens)
    assert torch.equal(apply_rules(x, r, hist[0]), torch.stack([apply_rules(x[:, t], r, hist[0]) for t in range(4)], 1))
    # other memory orders: transposed, every second column, expanded, one row without an axis
    xt = x.view(12, 29).t().contiguous().t()
    assert not xt.is_contiguous() and torch.equal(apply_rules(xt, r, flat, lens.view(12)), want)
    wide = torch.zeros(12, 58, device=cuda)
    wide[:, ::2] = x.view(12, 29)
    assert torch.equal(apply_rules(wide[:, ::2], r, flat, lens.view(12)), want)
    assert torch.equal(apply_rules(x[0, 0].expand(5, 29), r, hist[0]), apply_rules(x[0, 0], r, hist[0]).expand(5, 29))
    assert choose(x[0, 0], r, hist[0]).tokens.shape == ()
    # histories: a transposed one, one row for all
    ht = flat.t().contiguous().t()
    assert torch.equal(apply_rules(x.view(12, 29), r, ht, lens.view(12)), want)
    # gradients of an expanded row and of a transposed matrix arrive in its layout
    base = x[0, 0].clone().requires_grad_(True)
    tok = torch.arange(5, device=cuda)
    token_logprob(base.expand(5, 29), tok, r, hist[0]).sum().backward()
    parts = [torch.autograd.grad(token_logprob(b, tok[i], r, hist[0]), b)[0]
             for i in range(5) for b in [x[0, 0].clone().requires_grad_(True)]]
    assert torch.allclose(base.grad, torch.stack(parts).sum(0), rtol=0, atol=5 * 5 * U)


def test_no_rows(cuda):
    from dvae_amd.rules import TokenRules, apply_rules, choose, token_logprob
    b = torch.zeros(7, device=cuda, requires_grad=True)
    x = torch.zeros(0, 7, device=cuda, requires_grad=True)
    r = TokenRules(bias=b)
    with torch.no_grad():
        assert apply_rules(x, r).shape == (0, 7)
    got = choose(x, r, history=torch.zeros(0, 3, dtype=torch.int64, device=cuda), uniforms=torch.zeros(0, device=cuda))
    assert got.tokens.shape == (0,) and got.logprob.shape == (0,)
    lp = token_logprob(x, torch.zeros(0, dtype=torch.int64, device=cuda), r)
    dx, db = torch.autograd.grad(lp.sum(), [x, b])
    assert dx.shape == (0, 7) and torch.equal(db, torch.zeros(7, device=cuda))


def test_out_is_the_logits_or_apart_from_them(cuda):
    from dvae_amd.rules import TokenRules, apply_rules
    x = torch.zeros(4, 16, device=cuda)
    for out in (x[:, 1:9], x.view(2, 32)[:, :8], x[1:, :8]):
        with pytest.raises(ValueError):
            apply_rules(x[:out.shape[0], :8], TokenRules(), out=out)
    for out in (torch.zeros(4, 9, device=cuda), torch.zeros(4, 8, device=cuda, dtype=torch.float16),
                torch.zeros(8, 4, device=cuda).t(), torch.zeros(4, 8)):
        with pytest.raises(ValueError):
            apply_rules(x[:, :8], TokenRules(), out=out)


def test_offsets_beyond_32_bits(cuda):
    """Rows 1.2e9 elements apart: the third begins beyond 2^31 elements, and 2^32 bytes."""
    from dvae_amd.rules import TokenRules, apply_rules, choose, token_logprob
    ld, v = 1_200_000_000, 777
    base = torch.empty(2 * ld + v, dtype=torch.bfloat16, device=cuda)
    x = base.as_strided((3, v), (ld, 1))
    small = (torch.randn(3, v, generator=torch.Generator().manual_seed(0)) * 3).to(torch.bfloat16).to(cuda)
    x.copy_(small)
    u = torch.tensor([0.1, 0.5, 0.9], device=cuda)
    a, b = choose(x, uniforms=u), choose(small, uniforms=u)
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.logprob, b.logprob)
    r = TokenRules(bias=torch.randn(v, generator=torch.Generator().manual_seed(1)).to(cuda))
    assert torch.equal(apply_rules(x, r), apply_rules(small, r))
    assert torch.equal(token_logprob(x, a.tokens, r), token_logprob(small, a.tokens, r))
    apply_rules(x, r, out=x)
    assert torch.equal(x, apply_rules(small, r))


# ---- streams, graphs, autograd ----
def test_other_streams_and_two_calls_at_once(cuda):
    from dvae_amd.rules import choose
    case = Case(rows=40, vocab=9000, dtype="bf16", L=100, ragged=True, states=4, bias="shared", per_row=True, drawn=True, seed=6)
    x, kw, r = case.logits.to(cuda).contiguous(), case.kw(cuda), case.rules(cuda)
    t, u = case.temperature(cuda), case.u.to(cuda)
    want = choose(x, r, temperature=t, uniforms=u, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([choose(x, r, temperature=t, uniforms=u, **kw) for _ in range(3)])
    torch.cuda.synchronize()
    for one in got:
        for c in one:
            assert torch.equal(c.tokens, want.tokens) and torch.equal(c.logprob.nan_to_num(3.0), want.logprob.nan_to_num(3.0))


def test_captured_and_replayed(cuda):
    """Two graphs (a decision; a forward and backward pass), replayed in turn with new inputs and eager work between."""
    from dvae_amd.rules import choose, token_logprob
    case = Case(rows=12, vocab=9000, dtype="bf16", L=64, ragged=True, states=4, bias="shared", per_row=True, drawn=True, seed=7)
    x, kw, t, u = case.logits.to(cuda).contiguous(), case.kw(cuda), case.temperature(cuda), case.u.to(cuda)
    b, tok, g = case.bias.to(cuda).requires_grad_(True), case.tokens.to(cuda), case.g.to(cuda)
    r = case.rules(cuda, b)
    xg = x.clone().requires_grad_(True)

    def decide():
        return choose(x, r, temperature=t, uniforms=u, **kw)

    def train():
        lp = token_logprob(xg, tok, r, temperature=t, **kw)
        grads = torch.autograd.grad(lp, [xg, b], g)
        return (lp.detach(),) + grads                             # no graph of these leaves stays alive
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decide()
        train()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        c = decide()
    with torch.cuda.graph(g2):
        out = train()
    gen = torch.Generator().manual_seed(0)
    for i in range(4):
        fresh = (torch.randn(12, 9000, generator=gen) * 3).to(torch.bfloat16).to(cuda)
        with torch.no_grad():
            x.copy_(fresh)
            xg.copy_(fresh)
            u.copy_(torch.rand(12, generator=gen))
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        want, eager = decide(), train()
        assert torch.equal(c.tokens, want.tokens) and torch.equal(c.logprob.nan_to_num(3.0), want.logprob.nan_to_num(3.0))
        assert torch.equal(c.state, want.state)
        for a, e in zip(out, eager):
            assert torch.equal(a.nan_to_num(3.0), e.nan_to_num(3.0)), i


@pytest.mark.parametrize("shared", ["logits", "bias"])
def test_capture_beside_a_living_graph_is_refused(cuda, shared):
    """Of the same leaf, made on the default stream; without a gradient or after the graph's end a capture is none."""
    from dvae_amd._lib import DvaeError
    from dvae_amd.rules import TokenRules, token_logprob
    x, b = torch.randn(4, 300, device=cuda, requires_grad=True), torch.randn(300, device=cuda, requires_grad=True)
    y, c = torch.randn(4, 300, device=cuda, requires_grad=True), torch.randn(300, device=cuda, requires_grad=True)
    t = torch.tensor([0, 5, 299, -1], device=cuda)
    want = torch.autograd.grad(token_logprob(x, t, TokenRules(bias=b)).sum(), [x, b])
    alive = token_logprob(x if shared == "logits" else y, t, TokenRules(bias=b if shared == "bias" else c))
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(DvaeError, match="alive"):
            token_logprob(x, t, TokenRules(bias=b))
        with torch.no_grad():
            token_logprob(x, t, TokenRules(bias=b))
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(token_logprob(x, t, TokenRules(bias=b)), [x, b], torch.ones(4, device=cuda))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(got, want):
            assert torch.equal(u, v)


def test_capture_after_a_side_streams_living_graph(cuda):
    """A training step warmed up on a side stream, its last graph still alive, then captured: a trained bias accumulates."""
    from dvae_amd.rules import TokenRules, token_logprob
    x, b = torch.randn(4, 300, device=cuda), torch.randn(300, device=cuda, requires_grad=True)
    t = torch.tensor([0, 5, 299, -1], device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            b.grad = None
            loss = token_logprob(x, t, TokenRules(bias=b)).sum()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    want = b.grad.clone()
    torch.cuda.synchronize()
    b.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token_logprob(x, t, TokenRules(bias=b)).sum().backward()
    for _ in range(3):
        b.grad.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.grad, want)
    assert loss.grad_fn is not None


def test_changed_inputs_are_refused_by_the_backward_pass(cuda):
    from dvae_amd.rules import TokenRules, token_logprob
    x = torch.randn(3, 40, device=cuda, requires_grad=True)
    hist = torch.zeros(3, 4, dtype=torch.int64, device=cuda)
    rho = torch.full((3,), 1.5, device=cuda)
    for change in (hist, rho):
        lp = token_logprob(x, torch.zeros(3, dtype=torch.int64, device=cuda), TokenRules(repetition=rho), hist)
        change.add_(1)
        with pytest.raises(RuntimeError):
            lp.sum().backward()
    w = torch.ones(3, device=cuda, requires_grad=True)
    lp = token_logprob(x, torch.zeros(3, dtype=torch.int64, device=cuda))
    (d1,) = torch.autograd.grad((lp * w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d1.sum().backward()                                       # differentiable once


# ---- where the framework decides ----
def _dvae(cuda, N=7, C=6, mod=None):
    from argparse import Namespace
    import dvae_amd
    torch.manual_seed(3)
    m = dvae_amd.Dvae(Namespace(dataset_file=None, mod=mod, bidirectional=False, num_classes=C, max_seq=N, hidden_state_size=48))
    return m.to(cuda)


def _saved_elsewhere(cuda, bias_rows):
    """-> (leaves, call, junk): a call whose every argument is copied on the way in, its leaves, and what spoils its inputs."""
    from dvae_amd.rules import Grammar, TokenRules, token_logprob
    g = torch.Generator().manual_seed(17)
    rows, vocab, states = 6, 700, 3
    big = torch.randn(rows, vocab + 5, generator=g).to(cuda)
    history = torch.randint(0, vocab, (1, 40), generator=g, dtype=torch.int32).to(cuda).expand(rows, 40)
    lengths = torch.tensor([0, 1, 7, 39, 40, 90]).to(cuda)
    state = torch.tensor([0, 1, 2, 0, 1, 2]).to(cuda)
    tokens = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32).to(cuda)
    temperature = (0.5 + torch.rand(2 * rows, generator=g)).to(cuda)[::2]
    grammar = Grammar((torch.rand(states, vocab, generator=g) < 0.7).to(cuda))
    bias = torch.randn(*((rows,) if bias_rows else ()), 2 * vocab, generator=g).to(cuda).requires_grad_()
    big.requires_grad_()

    def call(big, bias):
        rules = TokenRules(1.2, 0.1, 0.2, bias[..., ::2], grammar)
        return token_logprob(big[:, :vocab] * 1.5, tokens, rules, history, lengths, state, temperature)

    def junk():                                     # temporaries that the call left behind are given out again
        for n in (rows, 2 * rows, vocab, rows * vocab, 40, 240):
            for t in (torch.float32, torch.int32, torch.int64):
                torch.full((n,), 3, dtype=t, device=cuda)
    return (big, bias), call, junk


@pytest.mark.parametrize("bias_rows", [False, True])
def test_hooks_of_saved_tensors(cuda, bias_rows):
    """Saved tensors that a hook stores on the host, or a checkpoint computes again, give the same bits."""
    leaves, call, junk = _saved_elsewhere(cuda, bias_rows)
    weight = torch.linspace(-1, 2, 6, device=cuda)
    lp = call(*leaves)
    want = torch.autograd.grad((lp * weight).sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        held = call(*leaves)
    junk()
    again = torch.utils.checkpoint.checkpoint(call, *leaves, use_reentrant=False)
    junk()
    for other in (held, again):
        assert torch.equal(other, lp)
        for a, b in zip(torch.autograd.grad((other * weight).sum(), leaves), want):
            assert torch.equal(a, b)


def test_a_hook_that_stored_the_logits_keeps_their_values(cuda):
    from dvae_amd.rules import token_logprob
    x = torch.linspace(-2, 2, 2 * 600, device=cuda).view(2, 600)
    t = torch.tensor([3, 599], device=cuda)
    want, = torch.autograd.grad(token_logprob(x.requires_grad_(), t).sum(), x)
    y = x.detach().clone().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        lp = token_logprob(y, t)
    with torch.no_grad():
        y.mul_(3.0)
    assert torch.equal(torch.autograd.grad(lp.sum(), y)[0], want)


def test_a_hook_that_stored_the_logits_frees_their_memory(cuda):
    from dvae_amd.rules import token_logprob
    x = torch.randn(64, 1 << 16, device=cuda, requires_grad=True)
    t = torch.arange(64, device=cuda)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        lp = token_logprob(x + 1.0, t)
    assert torch.cuda.memory_allocated() - before < x.numel() * 4
    want, = torch.autograd.grad(token_logprob(x + 1.0, t).sum(), x)
    assert torch.equal(torch.autograd.grad(lp.sum(), x)[0], want)


@pytest.mark.parametrize("mod", [None, "bn"])
def test_decoder_without_effective_rules_decides_as_before(cuda, mod):
    from dvae_amd.rules import TokenRules
    m = _dvae(cuda, mod=mod)
    z = torch.randn(33, 56, generator=torch.Generator().manual_seed(0)).to(cuda)
    e, t = m.decoder.predict(z)
    e2, t2 = m.decoder.predict(z, rules=TokenRules())
    assert torch.equal(e, e2) and torch.equal(t, t2)
    u = (torch.rand(33, 7, generator=torch.Generator().manual_seed(1)).to(cuda),
         torch.rand(33, 7, 7, generator=torch.Generator().manual_seed(2)).to(cuda))
    e, t = m.decoder.predict(z, uniforms=u)
    e2, t2 = m.decoder.predict(z, uniforms=u, rules=TokenRules())
    assert torch.equal(e, e2) and torch.equal(t, t2)


def test_decoder_under_a_grammar(cuda):
    from dvae_amd.rules import dag_rules
    m = _dvae(cuda)
    z = torch.randn(65, 56, generator=torch.Generator().manual_seed(0)).to(cuda)
    for stochastic in (False, True):
        edges, onehot = m.decoder.predict(z, stochastic, rules=dag_rules(6, 7, device=cuda), temperature=1.5)
        types = onehot.argmax(2)
        assert (onehot.sum(2) == 1).all() and ((onehot == 0) | (onehot == 1)).all()
        assert (types[:, 0] == 4).all() and (types[:, 6] == 5).all() and (types[:, 1:6] < 4).all()
        assert (edges == edges.tril(-1)).all()
    bn = _dvae(cuda, N=6, C=6, mod="bn")
    edges, onehot = bn.decoder.predict(z, True, rules=dag_rules(6, 6, "bn", device=cuda))
    inner = onehot[:, 1:5].argmax(2).sort(1).values
    assert (inner == torch.arange(4, device=cuda)).all()          # every variable once
    rep = bn.generation_eval(z=z, rules=dag_rules(6, 6, "bn", device=cuda), task_type="bn")
    assert 0.0 <= rep["validity"] <= 1.0


def test_decoder_where_the_rules_leave_nothing(cuda):
    """5 inner nodes, 4 types, none twice: the last inner node has no type left; the others are as they would be."""
    from dvae_amd.rules import TokenRules, dag_rules
    m = _dvae(cuda)
    g = dag_rules(6, 7, device=cuda).grammar
    z = torch.randn(9, 56, generator=torch.Generator().manual_seed(0)).to(cuda)
    edges, onehot = m.decoder.predict(z, rules=TokenRules(presence=math.inf, grammar=g))
    assert (onehot.sum(2) == torch.tensor([1.0, 1, 1, 1, 1, 0, 0], device=cuda)).all()   # no type, no step of the grammar
    assert torch.isfinite(edges).all()


def test_decoder_rows_of_their_own(cuda):
    """Per-latent settings: each latent decodes as it does alone with its setting."""
    from dvae_amd.rules import TokenRules
    m = _dvae(cuda)
    z = torch.randn(4, 56, generator=torch.Generator().manual_seed(0)).to(cuda)
    rep = torch.tensor([1.0, 2.0, 5.0, 50.0], device=cuda)
    bias = torch.linspace(-1, 1, 6, device=cuda)
    e, t = m.decoder.predict(z, rules=TokenRules(repetition=rep, bias=bias))
    for i in range(4):
        e1, t1 = m.decoder.predict(z[i:i + 1], rules=TokenRules(repetition=float(rep[i]), bias=bias))
        assert torch.equal(t[i], t1[0]) and torch.equal(e[i], e1[0])


def test_strings_under_a_grammar(cuda):
    from argparse import Namespace
    import dvae_amd
    from dvae_amd.rules import TokenRules, dag_rules
    sv = dvae_amd.Svae(Namespace(dataset_file=None, bidirectional=False)).to(cuda)
    g = torch.Generator().manual_seed(0)
    ts, es = torch.randn(50, 7, 8, generator=g).to(cuda), torch.randn(50, 7, 8, generator=g).to(cuda)
    plain = sv._predict_from_logits(ts, es)
    same = sv._predict_from_logits(ts, es, rules=TokenRules())
    assert all(torch.equal(a, b) for a, b in zip(plain, same))
    r = dag_rules(8, 8, start=1, device=cuda)
    for stochastic in (False, True):
        onehot, flags = sv._predict_from_logits(ts, es, is_stochastic=stochastic, rules=r, temperature=0.8)
        types = onehot.argmax(2)
        assert (onehot.sum(2) == 1).all() and (types[:, 6] == 7).all() and (types[:, :6] < 6).all()
    once = sv._predict_from_logits(ts, es, rules=TokenRules(presence=math.inf))[0].argmax(2)
    assert all(len(set(row)) == 7 for row in once.tolist())
    X = {"graph": torch.cat([plain[0], plain[1]], 2)}
    assert 0.0 <= sv.model_eval(X, 2, 2, rules=r)["recon_acc"] <= 1.0


def test_drawn_then_trained_on(cuda):
    """The run of all of them: graphs drawn under a grammar, the log-probability of their types through the decoder's own
    backward pass, the gradients clipped and stepped with -- against the same steps with the library's parts replaced by
    64-bit torch for the log-probability and by torch for clipping and Adam."""
    from dvae_amd.optim import FlatAdam, clip_grads, grad_norm
    from dvae_amd.rules import dag_rules, token_logprob
    m = _dvae(cuda)
    ref = _dvae(cuda)
    rules = dag_rules(6, 7, device=cuda)
    z = torch.randn(20, 56, generator=torch.Generator().manual_seed(0)).to(cuda)
    edges, onehot = m.decoder.predict(z, True, rules=rules)
    X = {"graph": edges, "node_encoding": onehot}
    tokens = onehot.argmax(2)
    state = torch.arange(7, dtype=torch.int32, device=cuda).expand(20, 7)
    reward = torch.randn(20, 1, generator=torch.Generator().manual_seed(1)).to(cuda)
    allowed = torch.zeros(7, 6, dtype=torch.bool, device=cuda)
    allowed[0, 4] = allowed[6, 5] = True
    allowed[1:6, :4] = True

    def loss(model, ours):
        _, scores = model.decoder(z, X)
        if ours:
            lp = token_logprob(scores, tokens, rules, state=state)
        else:
            y = scores.double().masked_fill(~allowed, -math.inf)
            lp = torch.log_softmax(y, 2).gather(2, tokens[..., None])[..., 0].float()
        return -(reward * lp).sum()
    a, b = loss(m, True), loss(ref, False)
    assert abs(float(a) - float(b)) <= 1e-5 * (abs(float(b)) + 140)
    a.backward()
    b.backward()
    ga = [p.grad for p in m.decoder.parameters() if p.grad is not None]
    gb = [p.grad for p in ref.decoder.parameters() if p.grad is not None]
    assert len(ga) == len(gb) > 0
    total = math.sqrt(sum(float(p.double().square().sum()) for p in gb))
    for p, q in zip(ga, gb):
        assert float((p - q).abs().max()) <= 2e-4 * max(float(q.abs().max()), 1e-3 * total)
    norm, coef = grad_norm(ga, total / 2)
    assert abs(float(norm) - total) <= 1e-4 * total and abs(float(coef) - 0.5) <= 1e-3
    opt = FlatAdam(m, lr=1e-2, max_norm=total / 2)
    opt.step()
    assert abs(float(opt.grad_norm) - total) <= 1e-4 * total
    clip_grads(gb, total / 2)
    topt = torch.optim.Adam(ref.parameters(), lr=1e-2)
    for p in ref.parameters():
        if p.grad is None:
            p.grad = torch.zeros_like(p)
    topt.step()
    # the first Adam step is lr * sign(g) where |g| >> eps: compare where the gradient is far from 0
    for (n, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        sure = q.grad.abs() > 1e-3 * float(q.grad.abs().max()) + 1e-6
        assert torch.allclose(p[sure], q[sure], rtol=0, atol=1e-5), n
