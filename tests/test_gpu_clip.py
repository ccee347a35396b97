"""GPU: global gradient norm and clipping against 64-bit sums.

Tolerances: squares and sums are doubles, so the norm is its exact value rounded once (2^-24, and 1e-12 for the sums'
order); coef is rounded once from a double; an output is the fp32 product (one rounding) of a rounded coef, rounded once
more to its type: 2 * 2^-24 + half a step of the type, and half a step of the smallest number."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
SIZES = [(1,), (3, 5), (0,), (8192,), (8193,), (127, 65), (1, 1, 1), (40000,), (2,), (511,), (70, 513)]


def make(sizes, dtypes, dev, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale * 10 ** (i % 3 - 1)).to(dtypes[i % len(dtypes)]).to(dev)
            for i, s in enumerate(sizes)]


def exact_norm(ts):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in ts))


def check(ts, outs, norm, before, max_norm):
    n = exact_norm(before)
    assert abs(float(norm) - n) <= n * (U + 1e-12)
    k = min(1.0, max_norm / (n + 1e-6))
    for t, o in zip(before, outs):
        want = t.double() * k
        h = torch.finfo(o.dtype).eps / 2
        err = (o.double() - want).abs()
        assert (err <= (2 * U + h + 1e-12) * want.abs() + TINY[o.dtype]).all()


@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES], ids=str)
def test_clip_in_place_and_into_others(cuda, dtypes, max_norm):
    from dvae_amd.optim import clip_grads, grad_norm
    ts = make(SIZES, dtypes, cuda)
    before = [t.clone() for t in ts]
    norm, coef = grad_norm(ts, max_norm)
    assert abs(float(coef) - min(1.0, max_norm / (exact_norm(before) + 1e-6))) <= 2 * U
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    for out_type in TYPES:
        outs = [torch.full_like(t, 7.0, dtype=out_type) for t in ts]
        check(ts, outs, clip_grads(ts, max_norm, out=outs), before, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check(ts, ts, clip_grads(ts, max_norm), before, max_norm)
    if max_norm == 1e9:
        assert all(torch.equal(a, b) for a, b in zip(ts, before))


@pytest.mark.parametrize("count", [1, 95, 96, 97, 300])
def test_many_tensors(cuda, count):
    from dvae_amd.optim import clip_grads
    ts = make([(1 + 37 * i % 911,) for i in range(count)], TYPES, cuda, seed=count)
    before = [t.clone() for t in ts]
    check(ts, ts, clip_grads(ts, 1.0), before, 1.0)


def test_views_that_begin_anywhere(cuda):
    """Tensors inside flat buffers at odd offsets, into views at other odd offsets; the gaps stay."""
    from dvae_amd.optim import clip_grads
    for dtype in TYPES:
        src = torch.randn(30000, device=cuda).to(dtype)
        dst = torch.full((30100,), 5.0, device=cuda)
        spans = [(1, 1001), (1003, 9300), (9301, 9302), (9305, 20000), (20001, 29999)]
        ts, outs = [src[a:b] for a, b in spans], [dst[a + 7:b + 7] for a, b in spans]
        before = [t.clone() for t in ts]
        check(ts, outs, clip_grads(ts, 1.0, out=outs), before, 1.0)
        covered = torch.zeros(30100, dtype=torch.bool, device=cuda)
        for a, b in spans:
            covered[a + 7:b + 7] = True
        assert (dst[~covered] == 5.0).all()
        keep = src.clone()
        clip_grads(ts, 1.0)
        mask = torch.zeros(30000, dtype=torch.bool, device=cuda)
        for a, b in spans:
            mask[a:b] = True
        assert torch.equal(src[~mask], keep[~mask])


def test_memory_orders(cuda):
    from dvae_amd.optim import clip_grads, grad_norm
    a = torch.randn(40, 30, device=cuda).t()
    b = torch.randn(2, 3, 4, 5, device=cuda).to(memory_format=torch.channels_last)
    before = [a.clone(), b.clone()]
    check([a, b], [a, b], clip_grads([a, b], 1.0), before, 1.0)
    assert a.stride() == (1, 30)
    o = torch.empty(40, 30, device=cuda).t()
    before = [a.clone()]
    check([a], [o], clip_grads([a], 0.25, out=[o]), before, 0.25)
    with pytest.raises(ValueError):
        grad_norm([torch.randn(4, 8, device=cuda)[:, :4]])


def test_extreme_magnitudes(cuda):
    """Squares that fp32 has no room for, either way."""
    from dvae_amd.optim import clip_grads
    for scale in (1e-30, 1e30):
        ts = [torch.full((1000,), scale, device=cuda), torch.full((24,), -scale, device=cuda)]
        before = [t.clone() for t in ts]
        check(ts, ts, clip_grads(ts, 1.0), before, 1.0)


def test_nan_and_infinity(cuda):
    from dvae_amd.optim import clip_grads, grad_norm
    ts = [torch.ones(5000, device=cuda), torch.ones(7, device=cuda)]
    ts[0][4321] = math.nan
    assert all(math.isnan(float(v)) for v in grad_norm(ts, 1.0))
    assert math.isnan(float(clip_grads(ts, 1.0))) and all(torch.isnan(t).all() for t in ts)
    ts = [torch.ones(5000, device=cuda), torch.ones(7, device=cuda)]
    ts[0][17] = -math.inf
    assert float(clip_grads(ts, 1.0)) == math.inf
    assert torch.isnan(ts[0][17]) and (ts[1] == 0).all() and (ts[0][18:] == 0).all()


def test_the_same_tensor_twice_is_refused(cuda):
    from dvae_amd import _lib
    from dvae_amd.optim import clip_grads, grad_norm
    t = torch.ones(100, device=cuda)
    for ts, out in (([t, t], None), ([t[:60], t[40:]], None), ([t[:40], t[40:80]], [t[20:60], t[60:]]),
                    ([t[:40]], [t[4:44]])):
        with pytest.raises(_lib.DvaeError):
            clip_grads(ts, 1.0, out=out)
    assert (t == 1).all()
    assert abs(float(grad_norm([t, t])[0]) - math.sqrt(200)) <= 15 * U        # reading it twice is a norm of both
    clip_grads([t[:50], t[50:]], 1.0)                                         # neighbours are fine
    assert abs(float(t.norm()) - 1.0) <= 1e-5


def test_autograd_sees_the_change(cuda):
    from dvae_amd.optim import clip_grads
    p = torch.ones(10, device=cuda, requires_grad=True)
    g = torch.ones(10, device=cuda)
    loss = (p * g).sum()
    clip_grads([g], 0.1)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_same_bits_on_every_call_and_stream(cuda):
    from dvae_amd.optim import clip_grads
    ts = make([(300000,), (77,), (1000, 333)], TYPES, cuda, seed=2)
    outs = [[torch.empty_like(t) for t in ts] for _ in range(4)]
    torch.cuda.synchronize()
    norms = []
    for i, o in enumerate(outs):
        with torch.cuda.stream(torch.cuda.Stream()):
            norms.append(clip_grads(ts, 1.0, out=o))
    torch.cuda.synchronize()
    for n, o in zip(norms[1:], outs[1:]):
        assert torch.equal(n, norms[0]) and all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_captured_and_replayed(cuda):
    from dvae_amd.optim import clip_grads
    ts = make([(30000,), (5,), (100, 333)], TYPES, cuda, seed=3)
    outs = [torch.empty(t.shape, device=cuda) for t in ts]
    clip_grads(ts, 1.0, out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grads(ts, 1.0, out=outs)
    for i in range(4):
        for t, f in zip(ts, make([(30000,), (5,), (100, 333)], TYPES, cuda, seed=10 + i, scale=1.0 + i)):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got, flat = norm.clone(), [o.clone() for o in outs]
        want = clip_grads(ts, 1.0, out=outs)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(flat, outs))


def _model(cuda):
    from argparse import Namespace
    import dvae_amd
    torch.manual_seed(5)
    return dvae_amd.Dvae(Namespace(dataset_file=None, mod=None, bidirectional=True, num_classes=6, max_seq=8,
                                   hidden_state_size=64)).to(cuda)


def test_flat_adam_with_a_largest_norm(cuda):
    """FlatAdam(max_norm) against the plain FlatAdam fed with gradients that clip_grads clipped: the same products, the
    same update, the same bits; p.grad itself stays unclipped."""
    import dvae_amd
    from dvae_amd.optim import FlatAdam, clip_grads, grad_norm
    a, b = _model(cuda), _model(cuda)
    oa, ob = FlatAdam(a, lr=1e-3, max_norm=1.0), FlatAdam(b, lr=1e-3)
    g, x = dvae_amd.synth.random_dags(10, 8, 6, 0.4, seed=3, chain=True)
    X = {'graph': g.to(cuda), 'node_encoding': x.to(cuda)}
    eps = torch.randn(10, 56, generator=torch.Generator().manual_seed(2)).to(cuda)
    for _ in range(3):
        a.loss_and_grad(X, eps=eps)
        b.loss_and_grad(X, eps=eps)
        raw = [p.grad.clone() for p in a.parameters()]
        oa.step()
        fe, fd = b._flat_grads()[:2]
        norm = clip_grads([fe, fd], 1.0)
        ob.step()
        assert float(norm) > 1.0 and torch.equal(norm, oa.grad_norm)
        assert all(torch.equal(p.grad, r) for p, r in zip(a.parameters(), raw))
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    assert oa.state_dict()['param_groups'][0].keys() == ob.state_dict()['param_groups'][0].keys()


@pytest.mark.parametrize("fused", [True, False])
def test_trainer_clips(cuda, fused):
    """Every step's norm is at most gradient_clip_val: seen by a torch Adam through p.grad, by FlatAdam through its norm."""
    import dvae_amd
    from dvae_amd.trainer import Trainer
    model = _model(cuda)
    g, x = dvae_amd.synth.random_dags(12, 8, 6, 0.4, seed=3, chain=True)
    model.train_loader = [{'graph': g[i:i + 6], 'node_encoding': x[i:i + 6]} for i in (0, 6)]
    model.val_loader = [None]
    seen = []
    made = model.configure_optimizers

    def configure(flat=False):
        (opt,), sched = made(flat=flat)
        step = opt.step

        def watched(*args):
            r = step(*args)
            n = opt.grad_norm if hasattr(opt, 'max_norm') else torch.stack([p.grad.double().norm() for p in model.parameters()]).norm()
            seen.append((type(opt).__name__, float(n), getattr(opt, 'max_norm', None)))
            return r
        opt.step = watched
        return [opt], sched
    model.configure_optimizers = configure
    Trainer(max_epochs=1, fused=fused, log=lambda r: None, gradient_clip_val=0.5).fit(model)
    assert len(seen) == 2
    if fused:
        assert all(n > 0.5 and m == 0.5 and kind == 'FlatAdam' for kind, n, m in seen)
    else:
        assert all(n <= 0.5 * (1 + 1e-5) for _, n, _ in seen)
