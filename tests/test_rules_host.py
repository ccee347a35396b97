"""Token rules and gradient clipping without a GPU: the grammar's tables, and every call that has to be refused."""
import ctypes
import math

import pytest
import torch

from dvae_amd import _lib, optim, rules
from dvae_amd.rules import Grammar, TokenRules


def test_grammar_packs_its_bits():
    gen = torch.Generator().manual_seed(0)
    for states, vocab in ((1, 1), (3, 31), (2, 32), (5, 33), (4, 100)):
        allowed = torch.rand(states, vocab, generator=gen) < 0.5
        allowed[0, vocab - 1] = True
        g = Grammar(allowed)
        assert g.masks.dtype == torch.int32 and g.masks.shape == (states, (vocab + 31) // 32) and g.next_state is None
        for s in range(states):
            for v in range(vocab):
                bit = (int(g.masks[s, v // 32]) >> (v % 32)) & 1
                assert bool(bit) == bool(allowed[s, v])
            for v in range(vocab, 32 * g.masks.shape[1]):
                assert not (int(g.masks[s, v // 32]) >> (v % 32)) & 1


def test_next_states_outside_the_table_stay_outside():
    allowed = torch.ones(3, 4, dtype=torch.bool)
    nxt = torch.tensor([[0, 1, 2, 3], [-7, 2 ** 40, -2 ** 40, 1], [0, 0, 0, 0]])
    g = Grammar(allowed, nxt)
    assert g.next_state.dtype == torch.int32
    assert g.next_state.tolist() == [[0, 1, 2, 3], [-1, 3, -1, 1], [0, 0, 0, 0]]
    small = torch.tensor([[0, -5, 7, 1]] * 3, dtype=torch.int32)
    assert Grammar(allowed, small).next_state.tolist() == small.tolist()


def test_grammar_refusals():
    ok = torch.ones(2, 3, dtype=torch.bool)
    for bad in (ok.int(), ok[0], torch.ones(0, 3, dtype=torch.bool), torch.ones(2, 0, dtype=torch.bool), [[True]]):
        with pytest.raises(ValueError):
            Grammar(bad)
    for nxt in (torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 3), torch.zeros(3, 2, dtype=torch.int64)):
        with pytest.raises(ValueError):
            Grammar(ok, nxt)
    for start in (-1, 2):
        with pytest.raises(ValueError):
            Grammar(ok, start=start)


def test_token_rules_refusals():
    for kw in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=math.inf), dict(repetition=math.nan),
               dict(frequency=math.inf), dict(frequency=math.nan), dict(presence=-math.inf), dict(presence=math.nan),
               dict(bias=torch.zeros(3, dtype=torch.float64)), dict(bias=torch.zeros(())), dict(bias=[0.0]),
               dict(repetition=torch.ones(3, dtype=torch.float16)),
               dict(presence=torch.ones(3, requires_grad=True)), dict(grammar=torch.ones(2, 3, dtype=torch.bool))):
        with pytest.raises(ValueError):
            TokenRules(**kw)
    assert not TokenRules(bias=torch.zeros(3), presence=math.inf).per_row()
    assert TokenRules(bias=torch.zeros(2, 3)).per_row() and TokenRules(frequency=torch.zeros(2)).per_row()


X = torch.zeros(4, 6)
G = Grammar(torch.ones(2, 6, dtype=torch.bool), torch.zeros(2, 6, dtype=torch.int32))
S = torch.zeros(4, dtype=torch.int32)
CALLS = [
    (X.double(), TokenRules(), {}),
    (X.int(), TokenRules(), {}),
    (torch.zeros(()), TokenRules(), {}),
    (torch.zeros(4, 0), TokenRules(), {}),
    (X, "rules", {}),
    (X, TokenRules(), dict(history=torch.zeros(4, 2))),
    (X, TokenRules(), dict(history=torch.zeros(3, 2, dtype=torch.int64))),
    (X, TokenRules(), dict(history=torch.zeros(4, 1, 2, dtype=torch.int64))),
    (X, TokenRules(), dict(history=torch.zeros(4, 2, dtype=torch.int16))),
    (X, TokenRules(), dict(lengths=S)),
    (X, TokenRules(), dict(history=torch.zeros(4, 2, dtype=torch.int64), lengths=S[:3])),
    (X, TokenRules(), dict(history=torch.zeros(4, 2, dtype=torch.int64), lengths=S.float())),
    (X, TokenRules(), dict(state=S)),
    (X, TokenRules(grammar=G), {}),
    (X, TokenRules(grammar=G), dict(state=S[:2])),
    (X, TokenRules(grammar=G), dict(state=S.float())),
    (X[:, :5], TokenRules(grammar=G), dict(state=S)),
    (X, TokenRules(bias=torch.zeros(5)), {}),
    (X, TokenRules(bias=torch.zeros(3, 6)), {}),
    (X, TokenRules(bias=torch.zeros(1, 4, 6)), {}),
    (X, TokenRules(repetition=torch.ones(3)), {}),
]


@pytest.mark.parametrize("i", range(len(CALLS)))
def test_refused_arguments(i):
    x, r, kw = CALLS[i]
    with pytest.raises(ValueError):
        rules.apply_rules(x, r, **kw)
    with pytest.raises(ValueError):
        rules.choose(x, r, **kw)
    with pytest.raises(ValueError):
        rules.token_logprob(x, torch.zeros(4, dtype=torch.int64), r, **kw)


def test_refused_temperatures_uniforms_tokens_and_outputs():
    for t in (0.0, -1.0, math.inf, math.nan, 1e-38, 1e38, torch.ones(3), torch.ones(4, dtype=torch.float64),
              torch.ones(4, requires_grad=True)):
        with pytest.raises(ValueError):
            rules.choose(X, TokenRules(), temperature=t)
        with pytest.raises(ValueError):
            rules.token_logprob(X, torch.zeros(4, dtype=torch.int64), temperature=t)
    with pytest.raises(ValueError):
        rules.apply_rules(X.clone().requires_grad_(True), TokenRules())
    # valid arguments, no GPU: no fallback
    for call in (lambda: rules.apply_rules(X, TokenRules()), lambda: rules.choose(X, uniforms=torch.zeros(4)),
                 lambda: rules.token_logprob(X, S)):
        with pytest.raises(_lib.DvaeError):
            call()


def test_dag_rules_tables():
    r = rules.dag_rules(8, 5)
    g = r.grammar
    assert (g.states, g.vocab, g.start) == (5, 8, 0) and r.presence == 0.0
    bits = [[bool((int(g.masks[s, 0]) >> v) & 1) for v in range(8)] for s in range(5)]
    assert bits[0] == [False] * 6 + [True, False] and bits[4] == [False] * 7 + [True]
    assert all(b == [True] * 6 + [False] * 2 for b in bits[1:4])
    assert g.next_state[:, 0].tolist() == [1, 2, 3, 4, 4]
    assert rules.dag_rules(10, 10, 'bn', start=1).presence == math.inf
    for bad in (dict(num_classes=2, max_seq=5), dict(num_classes=8, max_seq=1), dict(num_classes=8, max_seq=9, task_type='bn')):
        with pytest.raises(ValueError):
            rules.dag_rules(**bad)
    with pytest.raises(NotImplementedError):
        rules.dag_rules(8, 8, 'other')


def _q(**kw):
    q = _lib.DvaeRules()
    q.logits, q.rows, q.ld, q.vocab, q.dtype = 4096, 4, 16, 16, 0
    q.repetition = q.temperature = 1.0
    q.rows_per_history = 1
    for k, v in kw.items():
        setattr(q, k, v)
    return q


BAD_RULES = [dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(dtype=3), dict(logits=None),
             dict(ld=15), dict(repetition=0.0),
             dict(repetition=float("inf")), dict(frequency=float("nan")), dict(presence=float("nan")),
             dict(presence=float("-inf")), dict(temperature=0.0), dict(temperature=float("inf")),
             dict(temperature=9e-38), dict(temperature=1.1e37), dict(vocab=(1 << 27) + 1, ld=1 << 28),
             dict(history=4096, history_len=-1), dict(history=4096, history_len=2, history_ld=-1),
             dict(history=4096, history_len=2, rows_per_history=0), dict(mask=4096, states=1, mask_words=1),
             dict(mask=4096, states=0, mask_words=1, state=4096), dict(mask=4096, states=1, mask_words=0, state=4096),
             dict(rows=1 << 33), dict(rows=1 << 20, vocab=1 << 25, ld=1 << 25)]


@pytest.mark.parametrize("i", range(len(BAD_RULES)))
def test_c_abi_refuses_before_any_launch(i):
    """The descriptor is checked on the host first: the pointers here are never read."""
    lib = _lib.load()
    q, p = _q(**BAD_RULES[i]), ctypes.c_void_p(4096)
    assert lib.dvae_rules_apply(ctypes.byref(q), p, 1 << 31, None) == -1
    assert lib.dvae_rules_choose(ctypes.byref(q), None, None, p, p, None, p, None) == -1
    assert lib.dvae_rules_logprob(ctypes.byref(q), p, p, p, p, None) == -1
    assert lib.dvae_rules_logprob_bwd(ctypes.byref(q), p, p, p, p, 1 << 31, None, p, None) == -1
    assert lib.dvae_last_error()


def test_c_abi_refuses_missing_pointers():
    lib, p = _lib.load(), ctypes.c_void_p(4096)
    q = _q()
    r = ctypes.byref(q)
    assert lib.dvae_rules_apply(None, p, 16, None) == -1
    assert lib.dvae_rules_apply(r, None, 16, None) == -1
    assert lib.dvae_rules_apply(r, p, 15, None) == -1
    assert lib.dvae_rules_choose(r, None, None, None, p, None, p, None) == -1
    large = _q(vocab=4000, ld=4000)
    assert lib.dvae_rules_ws_bytes(r) == 0 and lib.dvae_rules_ws_bytes(ctypes.byref(large)) > 0
    assert lib.dvae_rules_choose(ctypes.byref(large), None, None, p, p, None, None, None) == -1
    assert lib.dvae_rules_logprob(ctypes.byref(large), p, p, p, None, None) == -1
    assert lib.dvae_rules_choose(r, None, p, p, p, None, p, None) == -1          # next without state_out
    assert lib.dvae_rules_choose(r, None, p, p, p, p, p, None) == -1             # next without a mask
    assert lib.dvae_rules_logprob(r, None, p, p, p, None) == -1
    assert lib.dvae_rules_logprob_bwd(r, p, p, p, None, 16, None, p, None) == -1
    assert lib.dvae_rules_logprob_bwd(r, p, p, p, p, 15, None, p, None) == -1
    assert lib.dvae_rules_logprob_bwd(r, p, p, p, p, 16, p, p, None) == -1       # d_bias without a bias
    # no rows: nothing to do, nothing read
    empty = _q(rows=0, logits=None)
    assert lib.dvae_rules_apply(ctypes.byref(empty), None, 16, None) == 0
    assert lib.dvae_rules_choose(ctypes.byref(empty), None, None, None, None, None, None, None) == 0
    assert lib.dvae_rules_logprob(ctypes.byref(empty), None, None, None, None, None) == 0
    assert lib.dvae_rules_ws_bytes(ctypes.byref(empty)) == 0


# ---- clipping ----
def test_clip_refusals():
    a = torch.zeros(4, 4)
    for bad in ([a.double()], [a, a.int()], [torch.zeros(4, 8)[:, :4]], [a.to_sparse()], ["x"],
                [torch.zeros(1, 4).expand(4, 4)]):
        with pytest.raises(ValueError):
            optim.grad_norm(bad)
        with pytest.raises(ValueError):
            optim.clip_grads(bad, 1.0)
    for m in (-1.0, math.nan):
        with pytest.raises(ValueError):
            optim.clip_grads([a], m)
    for out in ([], [a, a], [torch.zeros(4, 5)], [a.double()], [torch.zeros(4, 8)[:, :4]], [a.t()]):
        with pytest.raises(ValueError):
            optim.clip_grads([a], 1.0, out=out)
    with pytest.raises(ValueError):
        optim.clip_grads([a.clone().requires_grad_(True)], 1.0)
    with pytest.raises(_lib.DvaeError):
        optim.clip_grads([a], 1.0)
    assert float(optim.clip_grads([], 1.0)) == 0.0 and float(optim.clip_grads([None], 1.0)) == 0.0


def _t(*rows):
    t = (_lib.DvaeTensor * len(rows))()
    for d, (i, o, n, it, ot) in zip(t, rows):
        d.in_, d.out, d.n, d.in_type, d.out_type = i, o, n, it, ot
    return t


BAD_TENSORS = [
    [(4096, 4096, -1, 0, 0)], [(4096, 4096, 8, 3, 0)], [(4096, 8192, 8, 0, -1)], [(None, 4096, 8, 0, 0)],
    [(4096, None, 8, 0, 0)], [(4098, 8192, 8, 0, 0)], [(4097, 8192, 8, 1, 0)], [(4096, 8194, 8, 0, 0)],
    [(4096, 4096, 8, 1, 0)],                                           # its own output in another type
    [(4096, 4096, 8, 0, 0), (4096, 4096, 8, 0, 0)],                    # the same tensor twice
    [(4096, 4096, 8, 0, 0), (4112, 4112, 8, 0, 0)],                    # two tensors overlap by half
    [(4096, 8192, 8, 0, 0), (4096 + 512, 8192 + 28, 8, 0, 0)],         # two outputs overlap
    [(4096, 4100, 8, 0, 0)],                                           # an output over its own input, shifted
    [(4096, 8192, 8, 0, 0), (8192 + 16, 16384, 8, 0, 0)],              # an output over another input
]


@pytest.mark.parametrize("i", range(len(BAD_TENSORS)))
def test_clip_c_abi_refuses_before_any_launch(i):
    lib, p = _lib.load(), ctypes.c_void_p(1 << 20)
    t = _t(*BAD_TENSORS[i])
    assert lib.dvae_clip_grads(t, len(t), 1.0, p, p, None) == -1
    assert lib.dvae_last_error()


def test_clip_c_abi_pointers():
    lib, p = _lib.load(), ctypes.c_void_p(1 << 20)
    t = _t((4096, 4096, 8, 0, 0))
    assert lib.dvae_grad_norm(None, 1, 1.0, p, p, None) == -1
    assert lib.dvae_grad_norm(t, 1, 1.0, None, p, None) == -1
    assert lib.dvae_grad_norm(t, 1, 1.0, p, None, None) == -1
    assert lib.dvae_grad_norm(t, 1, -1.0, p, p, None) == -1
    assert lib.dvae_grad_norm(t, 1, float("nan"), p, p, None) == -1
    assert lib.dvae_clip_ws_bytes(-1) == 0 and lib.dvae_clip_ws_bytes(0) > 0
    assert lib.dvae_adam_step_scaled(p, p, None, p, p, 8, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None) == -1


def test_trainer_and_flat_adam_arguments():
    from dvae_amd.trainer import Trainer
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            Trainer(gradient_clip_val=bad)
    assert Trainer().gradient_clip_val == 0.0


def test_decoder_arguments():
    from argparse import Namespace
    import dvae_amd
    m = dvae_amd.Dvae(Namespace(dataset_file=None, mod=None, bidirectional=False, num_classes=6, max_seq=5,
                                hidden_state_size=32))
    z = torch.zeros(3, 56)
    with pytest.raises(ValueError):
        m.decoder.predict(z, rules=rules.dag_rules(6, 5), return_margin=True)
    with pytest.raises(ValueError):
        m.decoder.predict(z, temperature=0.5)
    with pytest.raises(ValueError):
        m.decoder.predict(z, rules=TokenRules(grammar=Grammar(torch.ones(2, 6, dtype=torch.bool))))
    with pytest.raises(ValueError):
        m.decoder.predict(z, rules=rules.dag_rules(7, 5))
    with pytest.raises(_lib.DvaeError):
        m.decoder.predict(z, rules=rules.dag_rules(6, 5))
    sv = dvae_amd.Svae(Namespace(dataset_file=None, bidirectional=False))
    ts, es = torch.zeros(2, 7, 8), torch.zeros(2, 7, 8)
    with pytest.raises(ValueError):
        sv._predict_from_logits(ts, es, temperature=0.5)
    with pytest.raises(ValueError):
        sv._predict_from_logits(ts[0], es[0], rules=TokenRules())


def test_sizes_that_a_c_int_does_not_hold():
    """Refused by the size alone: 2^32 + 5 is no 5 (views of one element: nothing is copied before)."""
    one, tok = torch.zeros(1, 1, dtype=torch.float16), torch.zeros(1, dtype=torch.int64)
    for vocab in (2 ** 27 + 1, 2 ** 31, 2 ** 32 + 5):
        x = one.expand(1, vocab)
        for call in (lambda: rules.apply_rules(x, TokenRules()), lambda: rules.choose(x), lambda: rules.token_logprob(x, tok)):
            with pytest.raises(ValueError, match="vocabulary"):
                call()
    for length in (2 ** 31, 2 ** 32 + 1):
        h = torch.zeros(1, 1, dtype=torch.int64).expand(1, length)
        for call in (lambda: rules.apply_rules(X[:1], TokenRules(), h), lambda: rules.choose(X[:1], history=h),
                     lambda: rules.token_logprob(X[:1], tok, history=h)):
            with pytest.raises(ValueError, match="history"):
                call()
    yes = torch.ones(1, 1, dtype=torch.bool)
    for shape in ((2 ** 31, 1), (1, 2 ** 27 + 1)):
        with pytest.raises(ValueError, match="too many"):
            Grammar(yes.expand(shape))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor would come back without its tangent: a derivative of 0 that nobody asked for."""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual, bias = fw.make_dual(X.clone(), torch.ones_like(X)), fw.make_dual(torch.zeros(6), torch.ones(6))
        for call in (lambda: rules.apply_rules(dual, TokenRules()), lambda: rules.apply_rules(X, TokenRules(bias=bias)),
                     lambda: rules.apply_rules(X, TokenRules(frequency=fw.make_dual(torch.zeros(4), torch.ones(4)))),
                     lambda: rules.apply_rules(X, TokenRules(), out=dual)):
            with pytest.raises(ValueError, match="dual"):
                call()
        with pytest.raises(_lib.DvaeError):            # plain tensors inside the level: on to the next check
            rules.apply_rules(X, TokenRules())


def test_out_over_an_argument():
    """A workgroup would read what another one has written.  (No GPU: the check of the device comes first, so stand in for it.)"""
    flat = torch.zeros(40)
    bias, rest = flat[10:16], flat[16:40].view(4, 6)
    setting, apart = flat[:4], flat[4:10]
    ids = torch.zeros(40, dtype=torch.int32)
    floats = ids.view(torch.float32)
    require, launch = rules.E._require_cuda, rules._Call.launch
    try:
        rules.E._require_cuda = lambda *a: None
        rules._Call.launch = lambda *a: None
        for out, r, kw in ((flat[:24].view(4, 6), TokenRules(bias=bias), {}), (flat[:24].view(4, 6), TokenRules(frequency=setting), {}),
                           (floats[:24].view(4, 6), TokenRules(), dict(history=ids[8:16].view(4, 2))),
                           (floats[:24].view(4, 6), TokenRules(), dict(history=ids[32:40].view(4, 2), lengths=ids[20:24])),
                           (floats[:24].view(4, 6), TokenRules(grammar=G), dict(state=ids[23:27]))):
            with pytest.raises(ValueError, match="out overlaps"):
                rules.apply_rules(X, r, out=out, **kw)
        assert rules.apply_rules(X, TokenRules(frequency=setting, bias=apart), out=rest) is rest          # neighbours
    finally:
        rules.E._require_cuda, rules._Call.launch = require, launch


def test_a_temperature_without_rules():
    """Refused wherever rules are optional: nothing would follow it."""
    from argparse import Namespace
    import dvae_amd
    from dvae_amd import dp
    m = dvae_amd.Dvae(Namespace(dataset_file=None, mod=None, bidirectional=False, num_classes=6, max_seq=5,
                                hidden_state_size=32))
    sv = dvae_amd.Svae(Namespace(dataset_file=None, bidirectional=False))
    z, ts, es = torch.zeros(3, 56), torch.zeros(2, 7, 8), torch.zeros(2, 7, 8)
    for kw in (dict(temperature=0.5), dict(temperature=torch.full((3,), 1.0)), dict(rules="dag")):
        for call in (lambda: m.decoder.predict(z, **kw), lambda: dp.predict_sharded(m.decoder, z, None, **kw),
                     lambda: m.generation_eval(z=z, **kw), lambda: sv._predict_from_logits(ts, es, **kw)):
            with pytest.raises(ValueError, match="rules"):
                call()


def test_trainer_leaves_an_optimizers_own_limit_alone(monkeypatch):
    """FlatAdam clips inside its step, at most to its own limit, and keeps it; any other optimizer's gradients are clipped for
    it, whatever attributes it has."""
    from dvae_amd import trainer
    clipped, seen = [], []
    monkeypatch.setattr(trainer, "clip_grads", lambda grads, limit: clipped.append((len(grads), limit)))
    flat = object.__new__(optim.FlatAdam)
    flat.step = lambda: seen.append(flat.max_norm)
    for own, want in ((None, 0.5), (0.1, 0.1), (3.0, 0.5)):
        flat.max_norm = own
        trainer.Trainer(gradient_clip_val=0.5)._step(flat)
        assert seen.pop() == want and flat.max_norm == own and not clipped

    class Other:
        max_norm, param_groups = 7.0, [{'params': [torch.zeros(2), torch.zeros(3)]}]

        def step(self):
            seen.append(self.max_norm)
    other = Other()
    trainer.Trainer(gradient_clip_val=0.5)._step(other)
    assert clipped == [(2, 0.5)] and seen == [7.0] and other.max_norm == 7.0
    trainer.Trainer()._step(other)
    assert len(clipped) == 1 and seen == [7.0, 7.0]
