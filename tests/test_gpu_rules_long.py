"""GPU: long histories over many rows, where segments are 4096 tokens long, against oracle/rules_ref.py with the bounds of
test_gpu_rules.py."""
import math

import numpy as np
import pytest
import torch

from oracle import rules_ref as R
from test_gpu_rules import Case, TINY, U, check_logprob, half, ident, log_z_tol, same_or_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [dict(rows=520, vocab=20001, L=5000, dtype="bf16", ragged=True, bias="shared", index=torch.int32),
                                   dict(rows=1100, vocab=8200, L=4097, dtype="fp32", states=3, per_row=True, pad=1),
                                   dict(rows=4200, vocab=4000, L=4500, dtype="fp16", junk=True)], ids=ident)
def test_long_histories(cuda, shape):
    """Rows of several segments, of three with a short last one, and of one (a wave decides it)."""
    from dvae_amd.rules import apply_rules, choose, token_logprob
    case = Case(seed=21, drawn=True, **shape)
    x, kw, temp = case.big.to(cuda)[:, :case.vocab], case.kw(cuda), case.temperature(cuda)
    got = apply_rules(x, case.rules(cuda), **kw)
    draw = choose(x, case.rules(cuda), temperature=temp, uniforms=case.u.to(cuda), **kw)
    best = choose(x, case.rules(cuda), temperature=temp, **kw)
    x = x.requires_grad_(True)
    lp = token_logprob(x, case.tokens.to(cuda), case.rules(cuda), temperature=temp, **kw)
    (dx,) = torch.autograd.grad(lp, x, case.g.to(cuda))
    some = list(range(0, case.nrows, case.nrows // 23)) + [case.nrows - 1]
    for r in some:
        y, _, _, t = case.row(r)
        same_or_close(got[r].double().cpu().numpy(), y,
                      (half(case.dtype) + U) * np.abs(np.where(np.isfinite(y), y, 0)) + TINY[case.dtype], "row %d" % r)
        for c, u in ((draw, float(case.u[r])), (best, None)):
            k, l = R.choose_row(y, t, u)
            assert int(c.tokens[r]) == k, (r, u)
            tol = U * abs(l) + 1e-11 + (0.0 if u is not None else log_z_tol(case, y, t)) if math.isfinite(l) else 0.0
            same_or_close(float(c.logprob[r]), l, tol, "row %d" % r)
    check_logprob(cuda, case, x, None, lp, dx, None, case.g, some)
