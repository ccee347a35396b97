"""Token decisions under rules: penalties for tokens a row's history holds, a bias, a grammar's mask (csrc/rules.hip).

The reference decides node types by a plain argmax or draw (Decoder.predict, dvae_model.py:282-291;
Svae._predict_from_logits, svae_model.py:112-131).  Here the same decision can be constrained, its log-probability read
and differentiated, for vocabularies of up to 2^27 tokens and fp32, bf16 and fp16 logits.  With c(v) how often the row's
history holds v:

    x1 = x / repetition if x > 0 else x * repetition, where c > 0
    x2 = x1 - frequency * c - presence * [c > 0]
    x3 = x2 + bias[v]
    x4 = x3 where the row's grammar state allows v, -inf elsewhere;   p = softmax(x4 / temperature)

``apply_rules`` returns x4, ``choose`` a token per row (greedy or drawn), ``token_logprob`` log p of given tokens with the
gradients of the logits and the bias.  ``Decoder.predict(rules=)``, ``Svae._predict_from_logits(rules=)`` and what calls
them (``model_eval``, ``generation_eval``) decide node types this way; ``dag_rules`` makes the rules of valid DAGs.

Shapes.  Logits are ``[..., V]``; the leading axes are the rows.  ``history`` is ``[..., L]`` (int32 / int64) over the first
of those axes (``[B, L]`` beside logits ``[B, T, V]``: the T rows of a sequence share its history; ``[L]``: all rows do);
``lengths`` (one per row) says how many of its tokens count, entries outside ``[0, V)`` never do.  Settings are a float for
all rows or an fp32 tensor with one per row.  Rows may lie anywhere in memory as long as a row's logits are adjacent (other
layouts are copied).  Everything is queued on the current stream of the logits' device.

A row whose rules leave nothing: token -1, log-probability -inf, no gradient.  A row that allows a NaN or a +inf, or whose
own temperature is not in [1e-37, 1e37]: token -1, log-probability NaN.
"""
import collections
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from . import engine as E
from ._lib import load

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}       # DVAE_F32 / DVAE_BF16 / DVAE_F16
_INDEX = (torch.int32, torch.int64)
_MAX_VOCAB, _INT_MAX = 2 ** 27, 2 ** 31 - 1                             # what csrc/rules.hip holds; what a C int does

Choice = collections.namedtuple("Choice", "tokens logprob state")


class Grammar:
    """A grammar as a table: ``allowed`` bool [S, V] -- state s allows token v -- and ``next_state`` int [S, V], the state
    after token v (optional; a value outside [0, S) is a state that allows everything).  ``start``: the state before the
    first token.  ``masks`` holds ``allowed`` as packed bits: bit v % 32 of word v // 32."""

    def __init__(self, allowed, next_state=None, start=0):
        if not torch.is_tensor(allowed) or allowed.dtype != torch.bool or allowed.dim() != 2 or 0 in allowed.shape:
            raise ValueError("Grammar: allowed must be a bool tensor [states, vocab]")
        self.states, self.vocab = (int(n) for n in allowed.shape)
        if self.vocab > _MAX_VOCAB or self.states > _INT_MAX:
            raise ValueError("Grammar: %d states of %d tokens are too many" % (self.states, self.vocab))
        if not 0 <= int(start) < self.states:
            raise ValueError("Grammar: start state %d of %d" % (int(start), self.states))
        self.start = int(start)
        # 32 tokens a word; as int32, where bit 31 is the sign: the sum of distinct powers of two wraps to the right word
        bits = torch.nn.functional.pad(allowed.int(), (0, -self.vocab % 32)).view(self.states, -1, 32)
        weight = torch.bitwise_left_shift(1, torch.arange(32, dtype=torch.int32, device=allowed.device))
        self.masks = (bits * weight).sum(2, dtype=torch.int32)
        self.next_state = None
        if next_state is not None:
            if not torch.is_tensor(next_state) or next_state.dtype not in _INDEX or next_state.shape != allowed.shape:
                raise ValueError("Grammar: next_state must be an int32 / int64 tensor [states, vocab]")
            if next_state.device != allowed.device:
                raise ValueError("Grammar: next_state is on %s, allowed on %s" % (next_state.device, allowed.device))
            if next_state.dtype != torch.int32:
                next_state = next_state.clamp(-1, self.states).to(torch.int32)
            self.next_state = next_state.contiguous()

    def to(self, device):
        g = object.__new__(Grammar)
        g.__dict__.update(self.__dict__)
        g.masks = self.masks.to(device)
        g.next_state = None if self.next_state is None else self.next_state.to(device)
        return g


class TokenRules:
    """What a decision follows: ``repetition`` (> 0, 1 = none), ``frequency``, ``presence`` (inf: no token twice) -- floats,
    or fp32 tensors with one value per row --, ``bias`` fp32 [V] or one row per row [..., V], and a ``Grammar``."""

    def __init__(self, repetition=1.0, frequency=0.0, presence=0.0, bias=None, grammar=None):
        for name, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            if torch.is_tensor(v):
                _per_row_check(v, name)
                continue
            v = float(v)
            if name == "repetition" and not (v > 0.0 and math.isfinite(v)):
                raise ValueError("TokenRules: repetition must be positive and finite, got %r" % v)
            if name == "frequency" and not math.isfinite(v):
                raise ValueError("TokenRules: frequency must be finite, got %r" % v)
            if name == "presence" and not v > -math.inf:
                raise ValueError("TokenRules: presence must be above -inf, got %r" % v)
        if bias is not None and (not torch.is_tensor(bias) or bias.dtype != torch.float32 or bias.dim() < 1):
            raise ValueError("TokenRules: bias must be an fp32 tensor [V] or [..., V]")
        if grammar is not None and not isinstance(grammar, Grammar):
            raise ValueError("TokenRules: grammar must be a Grammar")
        self.repetition, self.frequency, self.presence = repetition, frequency, presence
        self.bias, self.grammar = bias, grammar

    def per_row(self):
        """Whether any setting is one per row (such rules fit one set of rows only)."""
        return any(torch.is_tensor(v) for v in (self.repetition, self.frequency, self.presence)) or (
            self.bias is not None and self.bias.dim() > 1)

    def to(self, device):
        def move(v):
            return v.to(device) if torch.is_tensor(v) else v
        r = TokenRules(move(self.repetition), move(self.frequency), move(self.presence), move(self.bias))
        r.grammar = None if self.grammar is None else self.grammar.to(device)
        return r


def dag_rules(num_classes, max_seq, task_type='enas', start=0, device=None):
    """Rules under which a type string can be one of ``metrics.dag_validity``'s valid graphs (dataloader.py:57-88: node 0
    has the start type num_classes - 2, node max_seq - 1 the end type num_classes - 1, no other node either).  'bn': the
    variable nodes carry distinct types as well.  ``start``: the node of the first decision (1 for S-VAE strings, which
    leave the start node out)."""
    if task_type not in ('enas', 'bn'):
        raise NotImplementedError
    C, N = int(num_classes), int(max_seq)
    if C < 3 or N < 2:
        raise ValueError("dag_rules: at least 3 types and 2 nodes")
    if task_type == 'bn' and N > C:
        raise ValueError("dag_rules: %d variable nodes have no %d distinct types" % (N - 2, C - 2))
    allowed = torch.zeros(N, C, dtype=torch.bool)
    allowed[:, :C - 2] = True
    allowed[0] = allowed[N - 1] = False
    allowed[0, C - 2] = allowed[N - 1, C - 1] = True
    following = torch.arange(1, N + 1, dtype=torch.int32).clamp(max=N - 1).view(N, 1).repeat(1, C)
    rules = TokenRules(presence=math.inf if task_type == 'bn' else 0.0, grammar=Grammar(allowed, following, start))
    return rules if device is None else rules.to(device)


# ---------------------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------------------
def _per_row_check(t, name):
    if t.dtype != torch.float32:
        raise ValueError("%s: one value per row is an fp32 tensor, got %s" % (name, t.dtype))
    if t.requires_grad:
        raise ValueError("%s has no gradient: detach it" % name)


def _rows2d(t):
    """[..., n] -> [rows, n] with adjacent rows' elements; a view where the layout allows."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, n = t.shape
    s0, s1 = t.stride()
    if (n > 1 and s1 != 1) or (rows > 1 and s0 < n):
        t = t.contiguous()
    return t


class _Call:
    """The checked arguments of one call: the C descriptor `q` and the tensors behind its pointers."""

    def __init__(self, logits, rules, history, lengths, state, temperature):
        if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
            raise ValueError("logits must be an fp32, bf16 or fp16 tensor [..., V]")
        shape = logits.shape
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError("logits must have a vocabulary axis, got %s" % (tuple(shape),))
        if shape[-1] > _MAX_VOCAB:
            raise ValueError("a vocabulary of %d tokens: at most 2^27" % shape[-1])
        if rules is None:
            rules = TokenRules()
        elif not isinstance(rules, TokenRules):
            raise ValueError("rules must be a TokenRules")
        self.lead, self.V = lead, V = shape[:-1], shape[-1]
        self.rows = rows = math.prod(lead)
        self.index = index = logits.get_device()           # -1: the CPU
        self.device = logits.device
        self.logits = x = _rows2d(logits)
        q = _lib.DvaeRules(logits=x.data_ptr(), rows=rows, ld=x.stride(0) if rows > 1 else V, vocab=V,
                           dtype=_DTYPES[x.dtype], rows_per_history=1)
        self.tensors, self.fields = keep, fields = [], []  # behind q's pointers, besides logits and bias, and q's names for them
        if history is not None:
            if not isinstance(history, torch.Tensor) or history.dtype not in _INDEX or history.dim() < 1:
                raise ValueError("history must be an int32 / int64 tensor [..., L]")
            if history.shape[:-1] != lead[:history.dim() - 1]:
                raise ValueError("history %s does not go with the rows %s" % (tuple(history.shape), tuple(lead)))
            self._here(history, "history")
            L = history.shape[-1]
            if L > _INT_MAX:
                raise ValueError("a history of %d tokens: at most 2^31 - 1" % L)
            if L > 0 and rows > 0:
                h = history if history.dim() == 2 else history.reshape(-1, L)
                if L > 1 and h.stride(1) != 1:
                    h = h.contiguous()
                n = h.shape[0]
                q.history, q.history_len, q.history_ld = h.data_ptr(), L, h.stride(0) if n > 1 else 0
                q.history_i64 = h.dtype == torch.int64
                q.rows_per_history = rows // n
                keep.append(h)
                fields.append("history")
            if lengths is not None:
                self._per_row(lengths, "lengths", _INDEX)
                if lengths.dtype != torch.int32:
                    lengths = lengths.clamp(0, L).to(torch.int32)
                lengths = lengths.contiguous()
                q.lengths = lengths.data_ptr()
                keep.append(lengths)
                fields.append("lengths")
        elif lengths is not None:
            raise ValueError("lengths without a history")
        grammar = rules.grammar
        if grammar is not None:
            if grammar.vocab != V:
                raise ValueError("the grammar has %d tokens, the logits %d" % (grammar.vocab, V))
            if state is None:
                raise ValueError("a grammar needs the rows' state")
            masks = self._here(grammar.masks, "grammar")
            self._per_row(state, "state", _INDEX)
            if state.dtype != torch.int32:
                state = state.clamp(-1, grammar.states).to(torch.int32)
            state = state.contiguous()
            q.mask, q.mask_words, q.states, q.state = masks.data_ptr(), masks.shape[1], masks.shape[0], state.data_ptr()
            keep.extend((masks, state))
            fields.extend(("mask", "state"))
        elif state is not None:
            raise ValueError("state without a grammar")
        self.bias = None
        if rules.bias is not None:
            b = self._here(rules.bias, "bias")
            if b.shape[-1] != V or (b.dim() > 1 and b.shape[:-1] != lead):
                raise ValueError("bias %s does not go with logits %s" % (tuple(b.shape), tuple(shape)))
            if b.dim() == 1:
                self.bias = b if V == 1 or b.stride(0) == 1 else b.contiguous()
            else:
                self.bias = _rows2d(b)
                q.bias_ld = self.bias.stride(0) if rows > 1 else V
            q.bias = self.bias.data_ptr()
        q.repetition = self._setting(q, "repetition", rules.repetition)
        q.frequency = self._setting(q, "frequency", rules.frequency)
        q.presence = self._setting(q, "presence", rules.presence)
        q.temperature = t = self._setting(q, "temperature", temperature)
        if not 1e-37 <= t <= 1e37:
            raise ValueError("temperature must be in [1e-37, 1e37], got %r" % t)
        if index < 0:
            E._require_cuda(logits, "logits")
        self.q = q

    def _setting(self, q, name, v):
        if not isinstance(v, torch.Tensor):
            return float(v)
        _per_row_check(v, name)
        v = self._per_row(v, name, (torch.float32,)).contiguous()
        setattr(q, name + "_rows", v.data_ptr())
        self.tensors.append(v)
        self.fields.append(name + "_rows")
        return 1.0

    def _here(self, t, name):
        if t.get_device() != self.index:
            raise _lib.DvaeError("%s is on %s, the logits on %s" % (name, t.device, self.device))
        return t

    def _per_row(self, t, name, dtypes):
        if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.shape != self.lead:
            raise ValueError("%s must hold one value per row: a tensor %s of %s" %
                             (name, tuple(self.lead), " / ".join(str(d) for d in dtypes)))
        return self._here(t, name)

    def workspace(self):
        """-> (address or None, tensor): the tensor is to live until the launch is queued."""
        n = load().dvae_rules_ws_bytes(self.q)
        if not n:
            return None, None
        ws = E._workspace(n, self.device)
        return ws.data_ptr(), ws

    def launch(self, fn, *args):
        E._on_device(self.index, fn, self.q, *args)

    def elsewhere(self, logits, bias, *others):
        """-> (descriptor, tensors behind it) of the same call on copies of its tensors."""
        q = _lib.DvaeRules.from_buffer_copy(self.q)
        x = _rows2d(self._here(logits, "logits"))
        q.logits, q.ld = x.data_ptr(), x.stride(0) if self.rows > 1 else self.V
        keep = [x]
        if bias is not None:
            b = self._here(bias, "bias")
            b = b.contiguous() if b.dim() == 1 else _rows2d(b)
            q.bias = b.data_ptr()
            if b.dim() > 1:
                q.bias_ld = b.stride(0) if self.rows > 1 else self.V
            keep.append(b)
        for name, t in zip(self.fields, others):
            t = self._here(t, name).contiguous()
            setattr(q, name, t.data_ptr())
            if name == "history":
                q.history_ld = t.shape[1] if t.shape[0] > 1 else 0
            keep.append(t)
        return q, keep


def check_rules(rules, temperature, what):
    """For callers with optional rules, which decide plainly without them -- at temperature 1."""
    if rules is None:
        if torch.is_tensor(temperature) or temperature != 1.0:
            raise ValueError("%s: a temperature goes with rules" % what)
    elif not isinstance(rules, TokenRules):
        raise ValueError("%s: rules must be a TokenRules" % what)


def _address(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------------
# operators
# ---------------------------------------------------------------------------------------------------------------
def apply_rules(logits, rules, history=None, lengths=None, state=None, out=None):
    """-> x4 in the logits' type (one rounding).  ``out``: a tensor like the logits to write, which may be the logits
    themselves, but nothing else that the call reads; its rows must have adjacent elements.  No gradient: see
    ``token_logprob``."""
    if torch.is_grad_enabled() and torch.is_tensor(logits) and logits.requires_grad:
        raise ValueError("apply_rules has no gradient: detach the logits, or use token_logprob")
    if torch.is_grad_enabled() and isinstance(rules, TokenRules) and rules.bias is not None and rules.bias.requires_grad:
        raise ValueError("apply_rules has no gradient: detach the bias, or use token_logprob")
    if forward_ad._current_level >= 0:
        for t in (logits, out, *(vars(rules).values() if isinstance(rules, TokenRules) else ())):
            if torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("apply_rules has no gradient: its arguments must not be dual tensors")
    c = _Call(logits, rules, history, lengths, state, 1.0)
    if out is None:
        out = logits.new_empty(logits.shape)
        c.launch(load().dvae_rules_apply, out.data_ptr(), c.V)
        return out
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must be like the logits: %s %s on %s" % (tuple(logits.shape), logits.dtype, logits.device))
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError("out requires a gradient")
    o2 = out if out.dim() == 2 else out.view(-1, c.V)
    if c.rows and ((c.V > 1 and o2.stride(1) != 1) or (c.rows > 1 and o2.stride(0) < c.V)):
        raise ValueError("out: a row's elements must be adjacent")
    ld = o2.stride(0) if c.rows > 1 else c.V
    if c.rows and out.data_ptr() != c.logits.data_ptr():
        _apart(o2, c.logits, "out overlaps the logits")
    elif c.rows > 1 and ld != c.logits.stride(0):
        raise ValueError("out overlaps the logits")
    memory = out.untyped_storage().data_ptr()
    for t in (c.bias, *c.tensors):                            # read by every workgroup while others write
        if c.rows and t is not None and t.untyped_storage().data_ptr() == memory:
            _apart(o2, t, "out overlaps the bias, the history or a setting")
    c.launch(load().dvae_rules_apply, out.data_ptr(), ld)
    E._written([out])
    return out


def _span(t):
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _apart(a, b, text):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 < b1 and b0 < a1:
        raise ValueError(text)


def choose(logits, rules=None, history=None, lengths=None, state=None, temperature=1.0, uniforms=None):
    """One token per row -> ``Choice(tokens int64, logprob fp32, state int32 or None)``.

    Without ``uniforms`` the largest x4, the lowest index of equal ones.  With ``uniforms`` (fp32, one per row, in [0, 1)) the
    first token at which the running sum of p exceeds u (a p below 2^-990 of the largest is 0); either decision is the one of
    64-bit arithmetic.  ``logprob`` is log p of the token (detached; of a draw, and up to 128 tokens, from 64-bit sums, else
    greedily from fp32 ones as in ``token_logprob``: ordinarily off by a few 1e-7, by 4e-5 at most), ``state`` the grammar's next state where the grammar has
    ``next_state`` (a row without a token keeps its state)."""
    c = _Call(logits, rules, history, lengths, state, temperature)
    u = None
    if uniforms is not None:
        u = c._per_row(uniforms, "uniforms", (torch.float32,)).contiguous()
    tokens = logits.new_empty(c.lead, dtype=torch.int64)
    logprob = logits.new_empty(c.lead, dtype=torch.float32)
    following = nxt = None
    if rules is not None and rules.grammar is not None and rules.grammar.next_state is not None:
        nxt = c._here(rules.grammar.next_state, "grammar")
        following = logits.new_empty(c.lead, dtype=torch.int32)
    at, ws = c.workspace()
    c.launch(load().dvae_rules_choose, _address(u), _address(nxt), tokens.data_ptr(), logprob.data_ptr(),
             _address(following), at)
    return Choice(tokens, logprob, following)


class _LogprobFn(torch.autograd.Function):
    # Every tensor behind a pointer goes through save_for_backward, and nothing else keeps it: a change between forward and
    # backward is an error, and the backward pass (without retain_graph) frees it.  Logits and bias are saved as the call's
    # detached views, which stay on their memory if the caller gives its tensor another one (x.data = y).  Where hooks take saved
    # tensors (stored on the host, computed again by a checkpoint), what they give back is read instead.  The backward pass runs
    # on autograd's own thread, where Python is slowest: what it needs is at hand when the forward pass ends.
    @staticmethod
    def forward(ctx, call, logits, bias, tokens, *others):
        lib = load()
        ws, keep = call.workspace()
        logprob = logits.new_empty(call.rows, dtype=torch.float32)
        stat = logits.new_empty((call.rows, 2), dtype=torch.float64)
        at = tokens.data_ptr(), stat.data_ptr()
        call.launch(lib.dvae_rules_logprob, at[0], logprob.data_ptr(), at[1], ws)
        ctx.call, ctx.stat, ctx.at, ctx.fn = call, stat, at, lib.dvae_rules_logprob_bwd
        ctx.hooks = torch._C._autograd._top_saved_tensors_default_hooks(False) is not None
        ctx.save_for_backward(call.logits, call.bias, tokens, *others)
        call.logits = call.bias = None
        call.tensors = ()
        return logprob

    @staticmethod
    def backward(ctx, d_logprob):
        if torch.is_grad_enabled():                           # create_graph: the result refuses to be differentiated
            return once_differentiable(_LogprobFn._gradients)(ctx, d_logprob)
        return _LogprobFn._gradients(ctx, d_logprob)

    @staticmethod
    def _gradients(ctx, d_logprob):
        call = ctx.call
        logits, bias, tokens, *others = ctx.saved_tensors     # checks every saved tensor's version
        q, at = call.q, ctx.at
        if ctx.hooks:
            q, held = call.elsewhere(logits, bias, *others)
            tokens = call._here(tokens, "tokens").contiguous()
            at = tokens.data_ptr(), at[1]
        if d_logprob.dtype != torch.float32 or not d_logprob.is_contiguous():
            d_logprob = d_logprob.to(torch.float32).contiguous()
        d_logits = d_bias = ws = None
        _, want_logits, want_bias, *rest = ctx.needs_input_grad
        if want_logits:
            d_logits = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if want_bias:
            d_bias = torch.empty_like(bias, memory_format=torch.contiguous_format)
            ws, keep = call.workspace()
        E._on_device(call.index, ctx.fn, q, *at, d_logprob.data_ptr(), _address(d_logits), call.V, _address(d_bias), ws)
        return None, d_logits, d_bias, *([None] * len(rest))


def _on_default_stream(node, index):
    """Whether the stream is capturing and its backward pass would reach nodes (of the logits, of the bias) that this module
    first met on the default stream, which no capture can join (other streams it can)."""
    stream, found = torch._C._cuda_getCurrentRawStream(index), False
    for made, _ in node.next_functions[:2]:
        if made is not None and made.metadata.setdefault("dvae_stream", stream) == 0:
            found = True
    return found and stream != 0 and torch.cuda.is_current_stream_capturing()


def token_logprob(logits, tokens, rules=None, history=None, lengths=None, state=None, temperature=1.0):
    """log p of ``tokens`` (int32 / int64, one per row) under the rules, fp32, one per row; differentiable once with respect
    to the logits and the rules' bias.  A token outside [0, V) marks a row to ignore: 0 and no gradient.  A token the
    grammar forbids has -inf (and still the gradient -p / temperature of the allowed ones).

    Under capture into a HIP graph: autograd runs a leaf's accumulation on the stream where its first living graph was made,
    and a capture cannot wait for the default stream.  Where this function made that graph, it refuses: warm up on a side
    stream, end the eager graph before the capture, or use ``torch.no_grad()`` for a forward pass alone."""
    c = _Call(logits, rules, history, lengths, state, temperature)
    c._per_row(tokens, "tokens", _INDEX)
    tokens = (tokens if tokens.dtype == torch.int64 else tokens.to(torch.int64)).contiguous()
    x, b = c.logits, c.bias
    c.logits, c.bias = x.detach(), None if b is None else b.detach()
    lp = _LogprobFn.apply(c, x, b, tokens, *c.tensors)
    if lp.requires_grad and _on_default_stream(lp.grad_fn, c.index):
        lp = x = b = c = None                             # the error's traceback is not to keep this graph alive as well
        raise _lib.DvaeError("token_logprob: captured while a graph of the same tensor, made on the default stream, is alive")
    return lp if len(c.lead) == 1 else lp.view(c.lead)
