"""The optimizer of the reference's train step -- `torch.optim.Adam(self.parameters(), lr=1e-4)`
(dvae_model.py:471-475) -- over flat buffers: one HIP launch per module instead of torch's multi-tensor
launch over ~40 parameter tensors (110 us -> 35 us at hs=501; the step has nothing to overlap it with).

`FlatAdam` IS a `torch.optim.Optimizer`: `param_groups[0]['lr']` drives it (ReduceLROnPlateau works
unchanged) and its `state_dict()` has torch Adam's layout (`step`, `exp_avg`, `exp_avg_sq` per parameter), so
checkpoints move between the two.  The model's parameters become views of one flat buffer per module (same
`nn.Parameter` objects, same values), laid out like the flat gradient buffers `Dvae.loss_and_grad` fills.
"""
import array
import math

import torch

from . import engine as E

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}       # DVAE_F32 / DVAE_BF16 / DVAE_F16


def _flat_order(t):
    """Whether t's elements fill one stretch of memory, each once, in whatever order of its axes."""
    if t.is_contiguous():
        return True
    want = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda a: a[1]):
        if s != want:
            return False
        want *= n
    return True


def _flat_list(ts, what, name):
    """Dense fp32 / bf16 / fp16 tensors on one device -> (addresses, sizes, types, whether all are contiguous); each
    is one stretch of memory."""
    try:
        types = [_TYPES[t.dtype] for t in ts]
        plain = all([t.is_contiguous() for t in ts])
        if (plain or all([_flat_order(t) for t in ts])) and len({t.get_device() for t in ts}) <= 1:
            return [t.data_ptr() for t in ts], [t.numel() for t in ts], types, plain
    except (AttributeError, KeyError, RuntimeError):         # (a sparse tensor has no is_contiguous and no address)
        pass
    for i, t in enumerate(ts):           # which one it is
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.dtype not in _TYPES:
            raise ValueError("%s: %s %d must be a dense fp32, bf16 or fp16 tensor" % (what, name, i))
        if t.device != ts[0].device:
            raise ValueError("%s: %ss on %s and %s" % (what, name, ts[0].device, t.device))
        if not _flat_order(t):
            raise ValueError("%s: the elements of %s %d %s, strides %s, are not one stretch of memory" %
                             (what, name, i, tuple(t.shape), tuple(t.stride())))
    raise ValueError("%s: %ss must be tensors" % (what, name))


def _table(ins, outs):
    """An array of struct dvae_tensor: per tensor its two addresses, its size and (in one word) its two types."""
    (pi, n, ti, _), (po, _, to, _) = ins, outs
    table, types = array.array('q', bytes(32 * len(pi))), array.array('i', bytes(8 * len(pi)))
    types[0::2], types[1::2] = array.array('i', ti), array.array('i', to)
    table[0::4], table[1::4], table[2::4] = array.array('q', pi), array.array('q', po), array.array('q', n)
    table[3::4] = array.array('q', types.tobytes())
    return table


def _as_list(ts):
    return [ts] if isinstance(ts, torch.Tensor) else [t for t in ts if t is not None]


def _limit(max_norm, what):
    m = float(max_norm)
    if not m >= 0.0:
        raise ValueError("%s: max_norm must not be negative, got %r" % (what, m))
    return m


def grad_norm(grads, max_norm=math.inf):
    """-> (norm, coef): the norm of all gradients taken as one vector, and min(1, max_norm / (norm + 1e-6)), both scalars
    on the device (nothing waits for them).  ``grads``: tensors (fp32 / bf16 / fp16, each one stretch of memory; None is
    left out).  Sums are 64-bit in a fixed order: the same bits every time.  Neither result carries a gradient."""
    m = _limit(max_norm, "grad_norm")
    ts = _as_list(grads)
    ins = _flat_list(ts, "grad_norm", "gradient")
    if not ts:
        return torch.zeros(()), torch.ones(())
    E._require_cuda(ts[0], "gradient")
    out = torch.empty(2, device=ts[0].device)
    lib = E.load()
    ws = E._workspace(lib.dvae_clip_ws_bytes(len(ts)), ts[0].device)
    table = _table(ins, ins)
    E._on_device(ts[0].get_device(), lib.dvae_grad_norm, table.buffer_info()[0], len(ts), m, out.data_ptr(), ws.data_ptr())
    return out[0], out[1]


def clip_grads(grads, max_norm, out=None):
    """Scales the gradients so that their norm (see ``grad_norm``) is at most ``max_norm``, in place or, with ``out`` (a
    tensor for each, of any of the three types: contiguous as the gradient is, or of its shape and strides), into other
    tensors -- flat buffers, or single-precision copies of half-precision gradients.  Returns the norm before clipping, a
    scalar on the device.  The reference's Lightning Trainer has this as ``gradient_clip_val`` (train.py:41-47).  A NaN norm
    makes the gradients NaN; an infinite one makes them 0 (NaN where they were infinite)."""
    m = _limit(max_norm, "clip_grads")
    ts = _as_list(grads)
    ins = _flat_list(ts, "clip_grads", "gradient")
    os_, outs = ts, ins
    if out is not None:
        os_ = _as_list(out)
        if len(os_) != len(ts):
            raise ValueError("clip_grads: %d outputs for %d gradients" % (len(os_), len(ts)))
        outs = _flat_list(os_, "clip_grads", "output")
        if outs[1] != ins[1] or (ts and os_[0].get_device() != ts[0].get_device()):
            raise ValueError("clip_grads: outputs unlike the gradients: sizes %s for %s" % (outs[1], ins[1]))
        for i, (t, o) in enumerate(() if ins[3] and outs[3] else zip(ts, os_)):
            if not (t.is_contiguous() and o.is_contiguous()) and (t.shape != o.shape or any(
                    n > 1 and a != b for n, a, b in zip(t.shape, t.stride(), o.stride()))):
                raise ValueError("clip_grads: output %d is laid out unlike its gradient" % i)
    if torch.is_grad_enabled() and any([o.requires_grad for o in os_]):
        raise ValueError("clip_grads: an output that requires a gradient is not written in place")
    if not ts:
        return torch.zeros(())
    E._require_cuda(ts[0], "gradient")
    norm = torch.empty(2, device=ts[0].device)
    lib = E.load()
    ws = E._workspace(lib.dvae_clip_ws_bytes(len(ts)), ts[0].device)
    table = _table(ins, outs)
    E._on_device(ts[0].get_device(), lib.dvae_clip_grads, table.buffer_info()[0], len(ts), m, norm.data_ptr(), ws.data_ptr())
    E._written(os_)
    return norm[0]


class FlatAdam(torch.optim.Optimizer):
    """``max_norm`` (also an attribute, changeable between steps; None = no clipping): a step's update is that of gradients
    clipped to this norm.  ``p.grad`` keeps the gradients as they came -- the update kernel scales them as it reads them --
    and ``grad_norm`` the last clipped step's norm (a scalar on the device)."""

    def __init__(self, model, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, max_norm=None):
        self.max_norm = None if max_norm is None else _limit(max_norm, "FlatAdam")
        self.grad_norm = None
        enc_p, dec_p = model.encoder.hip_params(), model.decoder.hip_params()
        every = enc_p + dec_p
        if len({id(p) for p in every}) != len(every):
            raise ValueError("FlatAdam: modules share parameters (same_mapper_gater); use torch.optim.Adam")
        if {id(p) for p in every} != {id(p) for p in model.parameters()}:
            raise ValueError("FlatAdam: the model has parameters outside encoder / decoder")
        for p in every:
            if not p.is_cuda or p.dtype != torch.float32:
                raise ValueError("FlatAdam: fp32 parameters on a GPU")
        super().__init__(every, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._model = model
        self._t = 0
        self._mods = []
        with torch.no_grad():
            for plist in (enc_p, dec_p):
                flat = torch.cat([p.detach().reshape(-1) for p in plist])
                m, v = torch.zeros_like(flat), torch.zeros_like(flat)
                o = 0
                for p in plist:
                    n = p.numel()
                    p.data = flat[o:o + n].view_as(p)           # same Parameter object, storage inside `flat`
                    self.state[p] = {'step': torch.tensor(0.0), 'exp_avg': m[o:o + n].view_as(p),
                                     'exp_avg_sq': v[o:o + n].view_as(p)}
                    o += n
                self._mods.append((plist, flat, m, v))

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        g = self.param_groups[0]
        fe, fd, ve, vd = self._model._flat_grads()
        self._t += 1
        lib = E.load()
        stream = E._stream()
        for (plist, flat, m, v), fg, views in zip(self._mods, (fe, fd), (ve, vd)):
            # loss_and_grad leaves p.grad as views of the flat gradient buffer; gradients from autograd are copied in
            for p, gv in zip(plist, views):
                if p.grad is None:
                    gv.zero_()
                elif p.grad.data_ptr() != gv.data_ptr():
                    gv.copy_(p.grad)
        coef = None
        if self.max_norm is not None:
            self.grad_norm, coef = grad_norm((fe, fd), self.max_norm)
        for (plist, flat, m, v), fg in zip(self._mods, (fe, fd)):
            rest = (E._ptr(m), E._ptr(v), flat.numel(), float(g['lr']), float(g['betas'][0]), float(g['betas'][1]),
                    float(g['eps']), float(g['weight_decay']), self._t, stream)
            if coef is None:
                E.check(lib.dvae_adam_step(E._ptr(flat), E._ptr(fg), *rest))
            else:
                E.check(lib.dvae_adam_step_scaled(E._ptr(flat), E._ptr(fg), E._ptr(coef), *rest))
        return loss

    def state_dict(self):
        for st in self.state.values():
            st['step'] = torch.tensor(float(self._t))
        return super().state_dict()

    def load_state_dict(self, state_dict):
        views = {id(p): (st['exp_avg'], st['exp_avg_sq']) for p, st in self.state.items()}
        super().load_state_dict(state_dict)
        steps = set()
        with torch.no_grad():
            for p, st in self.state.items():
                m, v = views[id(p)]
                m.copy_(st['exp_avg'])
                v.copy_(st['exp_avg_sq'])
                steps.add(int(float(st['step'])))
                st['exp_avg'], st['exp_avg_sq'] = m, v
        if len(steps) > 1:
            raise ValueError("FlatAdam: parameters with different step counts")
        self._t = steps.pop() if steps else 0
