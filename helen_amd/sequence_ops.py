"""Sequence operators on the MI355X: the gated delta rule (whole sequences, forward and backward, and single tokens over a
pool of states) and layer norm (forward and backward).

They stand beside HelenEngine.chunk_forward, the GRU layer with a carried hidden state: torch tensors in, torch tensors out,
all compute in libhelen_hip.so (include/helen_hip.h), asynchronous on the current stream of the tensors' device.  Gradients
are calls of their own; `DeltaRule` and `LayerNorm` tie them into torch's autograd.  The plain calls record nothing: while
gradients are recorded they refuse inputs that require one.

A call keeps nothing: workspaces come from torch's allocator, so calls on several streams may run at once and a call may be
captured into a graph.  Nothing here waits for the device.

Outputs may not overlap inputs or themselves; the exception is layer_norm's `out`, which may be `x`.  What a call writes in place
(`out`, a pool of states) counts as modified for autograd, and may not require a gradient itself while gradients are recorded.
"""
import ctypes
import functools
import struct

import torch

from . import _lib

_TYPES = {torch.float32: _lib.HELEN_TYPE_FP32, torch.bfloat16: _lib.HELEN_TYPE_BF16, torch.float16: _lib.HELEN_TYPE_FP16}

# The descriptions of include/helen_hip.h in native layout: packed in one go, a quarter of the time of setting a ctypes
# structure's fields one by one (a single-token call is shorter on the GPU than on the host).
_RULE = struct.Struct("@N2i 4i 2i i f P 3P 2P 10q P P 2q P P 2q P 3P 3P".replace(" ", ""))
_STEP = struct.Struct("@N2i 4i 2i f P 3P 2P 10q P q P 2q".replace(" ", ""))
_NORM = struct.Struct("@N2i i i q f P q 2P P q 2P P q P q 2P".replace(" ", ""))


def _fail(message):
    raise ValueError(message)


def _gpu_index(name, t):
    """The device of a call's first tensor."""
    if not isinstance(t, torch.Tensor):
        _fail("%s must be a torch tensor" % name)
    device = t.get_device()
    if device < 0:
        raise RuntimeError("%s is not on a GPU: the sequence operators need one, there is no CPU fallback" % name)
    return device


def _same_gpu(name, t, device):
    if not isinstance(t, torch.Tensor):
        _fail("%s must be a torch tensor" % name)
    at = t.get_device()
    if at != device:
        if at < 0:
            raise RuntimeError("%s is not on a GPU: the sequence operators need one, there is no CPU fallback" % name)
        _fail("%s is on GPU %d, the other tensors on %d" % (name, at, device))


_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _inner(t, bytes_=0):
    """`t` with a contiguous last dimension and, where `bytes_` is given, base and strides that are multiples of it; a copy if
    it has to be one."""
    strides = t.stride()
    if strides[-1] != 1 and t.numel() and t.shape[-1] != 1:
        return t.contiguous()
    if bytes_:
        size = t.element_size()
        if t.data_ptr() % bytes_ or strides[0] > 1 << 24 or any(s * size % bytes_ for s in strides[:-1]):
            return t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else t.contiguous()
    return t


def _like(t):
    """A new contiguous tensor of t's shape and type (empty_like is the cheapest allocation a call can make)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


_wrote = torch.autograd.graph.increment_version      # (writes through a pointer are not seen by autograd otherwise)


_requires = torch._C._any_requires_grad if hasattr(torch._C, "_any_requires_grad") else (
    lambda *inputs: any(getattr(t, "requires_grad", False) for t in inputs))


def _recorded(*inputs):
    """Whether autograd records a call on these inputs."""
    return torch.is_grad_enabled() and _requires(*inputs)


def _outside(what, use, *written):
    """Refuses a call that autograd cannot follow: it would cut an input's graph without a word, or take what is written for the
    result of what made it."""
    if _requires(*written):
        raise RuntimeError("what %s writes requires a gradient and is written in place: call it under torch.no_grad(), or pass a "
                           "tensor that does not" % what)
    raise RuntimeError("%s records no gradients and an input requires one: %s under torch.no_grad()" % (what, use))


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _heads(q, k, v, g, beta):
    """Types, devices and shapes of a call's tokens: -> (device, type, tokens, heads_k, heads_v, width_k, width_v)."""
    device = _gpu_index("q", q)
    _same_gpu("k", k, device)
    _same_gpu("v", v, device)
    _same_gpu("g", g, device)
    _same_gpu("beta", beta, device)
    dtype = q.dtype
    code = _TYPES.get(dtype)
    if code is None:
        _fail("q is %s: float32, bfloat16 or float16 are supported" % dtype)
    if k.dtype != dtype or v.dtype != dtype:
        _fail("q, k, v are %s, %s, %s: one type is needed" % (dtype, k.dtype, v.dtype))
    if g.dtype != torch.float32 or beta.dtype != torch.float32:
        _fail("g and beta must be float32")
    shape, v_shape = q.shape, v.shape
    if len(shape) != 3 or len(v_shape) != 3:
        _fail("q, k, v must be [tokens, heads, width]")
    if k.shape != shape:
        _fail("k is %s, q %s" % (tuple(k.shape), tuple(shape)))
    n, hk, dk = shape
    nv, hv, dv = v_shape
    if nv != n:
        _fail("v has %d tokens, q %d" % (nv, n))
    if g.shape != v_shape[:2] or beta.shape != v_shape[:2]:
        _fail("g and beta must be [%d, %d]: they are %s and %s" % (n, hv, tuple(g.shape), tuple(beta.shape)))
    if dk not in (64, 128):
        _fail("width %d of q and k: 64 and 128 are supported" % dk)
    if dv not in (64, 128, 192, 256):
        _fail("width %d of v: 64, 128, 192 and 256 are supported" % dv)
    if hk < 1 or hv < 1 or hv % hk:
        _fail("%d value heads do not share %d key heads evenly" % (hv, hk))
    if n >= 2 ** 31:
        _fail("%d tokens in one call" % n)
    return device, code, n, hk, hv, dk, dv


def _state(name, t, shape, device):
    if t is None:
        return None
    _same_gpu(name, t, device)
    if t.dtype != torch.float32 or tuple(t.shape) != shape:
        _fail("%s must be float32 %s" % (name, shape))
    return t.contiguous()


def _output(name, t, shape, dtype, device):
    _same_gpu(name, t, device)
    if t.dtype != dtype or tuple(t.shape) != shape:
        _fail("%s must be %s %s" % (name, dtype, shape))
    if t.numel() and t.stride(-1) != 1:
        _fail("%s must have a contiguous last dimension" % name)
    if not t.is_contiguous():
        reach = 0                         # of the dimensions with smaller strides
        for stride, size in sorted(zip(t.stride(), t.shape)):
            if size > 1:
                if stride <= reach:
                    _fail("the elements of %s overlap" % name)
                reach += stride * (size - 1)
    return t


@functools.lru_cache(maxsize=1024)
def _rule_bytes(code, hk, hv, dk, dv, tokens, sequences):
    """Workspaces of a call of these sizes: forward, forward that keeps, backward."""
    op = _lib.HelenDeltaRuleC()
    op.struct_size = ctypes.sizeof(op)
    op.dtype, op.heads_k, op.heads_v, op.width_k, op.width_v, op.tokens, op.sequences = code, hk, hv, dk, dv, tokens, sequences
    op.offsets = 1       # (lengths may differ; not read)
    got = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(_lib.load().helen_delta_rule_bytes(ctypes.byref(op), *(ctypes.byref(x) for x in got)))
    return tuple(int(x.value) for x in got)


class _Call(object):
    """A checked delta rule call: what its C description is packed from, and the tensors it points into."""

    def __init__(self, q, k, v, g, beta, scale, initial_state, offsets):
        self.sizes = device, code, n, hk, hv, dk, dv = _heads(q, k, v, g, beta)
        self.device, self.dtype, self.tokens, self.hv, self.dv = device, q.dtype, n, hv, dv
        self.q, self.k, self.v = _inner(q, 16), _inner(k, 16), _inner(v, 16)
        self.g, self.beta = g, beta
        self.whole = True                  # every row belongs to a sequence, as far as the host can tell
        sequences = 1
        if offsets is not None:
            if isinstance(offsets, (list, tuple)):
                offsets = torch.tensor(offsets, dtype=torch.int64)
            if not (isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.numel() >= 2
                    and offsets.dtype in (torch.int32, torch.int64)):
                _fail("offsets must be one row of at least two int32 / int64")
            sequences = offsets.numel() - 1
            self.whole = False
            if offsets.is_cuda:
                _same_gpu("offsets", offsets, device)
            else:
                at = offsets.tolist()
                if at[0] != 0 or at[-1] > n or any(a > b for a, b in zip(at, at[1:])):
                    _fail("offsets must ascend from 0 to at most %d" % n)
                self.whole = at[-1] == n
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("offsets on the host cannot be captured into a graph: pass them on the GPU")
                offsets = offsets.to(torch.int32).pin_memory().to(q.device, non_blocking=True)
            if offsets.dtype != torch.int32 or not offsets.is_contiguous():
                offsets = offsets.to(torch.int32).contiguous()
        self.offsets = offsets
        self.sequences = sequences
        self.state_shape = (sequences, hv, dk, dv)
        self.initial = _state("initial_state", initial_state, self.state_shape, device)
        self.scale = dk ** -0.5 if scale is None else float(scale)
        self.work = _rule_bytes(code, hk, hv, dk, dv, n, sequences)

    def pack(self, o=None, final=None, zero_tail=0, d_o=None, d_final=None, grads=(None,) * 6):
        device, code, n, hk, hv, dk, dv = self.sizes
        q, k, v, g, beta = self.q, self.k, self.v, self.g, self.beta
        qs, ks, vs, gs, bs = q.stride(), k.stride(), v.stride(), g.stride(), beta.stride()
        os = o.stride() if o is not None else (0, 0)
        ds = d_o.stride() if d_o is not None else (0, 0)
        return _RULE.pack(_RULE.size, device, code, hk, hv, dk, dv, n, self.sequences, zero_tail, self.scale,
                          _ptr(self.offsets), q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                          qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], gs[0], gs[1], bs[0], bs[1],
                          _ptr(self.initial), _ptr(o), os[0], os[1], _ptr(final), _ptr(d_o), ds[0], ds[1], _ptr(d_final),
                          *map(_ptr, grads))

    def forward(self, o, keep, zero_tail=0):
        """-> (final_state, workspace); `o` None computes the states alone."""
        final = self.q.new_empty(self.state_shape, dtype=torch.float32)
        size = self.work[1 if keep else 0]
        work = self.q.new_empty(size, dtype=torch.uint8)
        rc = _lib.load().helen_delta_rule_forward(self.pack(o, final, zero_tail), int(keep), work.data_ptr(), size,
                                                  _stream(self.device))
        if rc:
            _lib.check(rc)
        return final, work


def delta_rule(q, k, v, g, beta, scale=None, initial_state=None, offsets=None, out=None, keep=False):
    """The gated delta rule over whole sequences.  Per value head a state S [width_k, width_v] and per token

        u = beta (v - e^g S^T k),    S <- e^g S + k u^T,    o = scale S^T q

    q, k [tokens, heads_k, width_k], v [tokens, heads_v, width_v] of one type (float32, bfloat16, float16), g (log decay) and
    beta float32 [tokens, heads_v]; value heads h of a group share key head h // (heads_v // heads_k).  Any strides; what is
    not 16-byte aligned with a contiguous last dimension is copied.  width_k 64 or 128, width_v 64, 128, 192 or 256.
      scale          default width_k ** -0.5
      initial_state  float32 [sequences, heads_v, width_k, width_v]; default zero
      offsets        int [sequences + 1]: sequence i is rows offsets[i] .. offsets[i + 1] (default: one sequence).  On the host
                     (list, CPU tensor) they are checked; on the GPU they must ascend from 0 to at most `tokens`: others give
                     wrong values, but no access out of range
      out            where o goes (any strides with a contiguous last dimension); rows behind the last sequence are left as
                     they are there, and zero in a fresh o
      keep           True: also return what delta_rule_backward needs of this call: per 64 tokens and at widths of 128
                     169 KB a value head (states, errors and triangles in float32 or three bf16 terms) and 84 KB a key head in
                     bf16 (148 in fp16, 212 in float32); 32 sequences of 1000 tokens with 4 / 8 heads in bf16 keep 921 MB where
                     q, k and v are 131.  The backward call takes 96 KB a value head more while it runs
    -> (o, final_state) or (o, final_state, saved).  All arithmetic is float32-class whatever the type of q, k, v: o is the float32
    result rounded once, states are float32.

    g is a decay: at most 0, -inf included (it forgets the state).  Positive values are taken as they are as long as e to their sum
    over 64 tokens is a float32.  (A NaN or an infinity in an initial state is not forgotten.)  Tokens are worked on in chunks of 64 (from the sequence's start): a NaN or an infinity in a
    token's q, k, v, g or beta reaches the results of its whole chunk, earlier tokens included, and what follows it, in its own
    sequence and heads; other sequences and heads stay as they are."""
    if _recorded(q, k, v, g, beta, initial_state, out):
        _outside("delta_rule", "use DeltaRule.apply, or call it", out)
    call = _Call(q, k, v, g, beta, scale, initial_state, offsets)
    shape = (call.tokens, call.hv, call.dv)
    if out is None:
        o, tail = _like(v), 0 if call.whole else 1
    else:
        o, tail = _output("out", out, shape, call.dtype, call.device), 0
    final, work = call.forward(o, keep, tail)
    if out is not None:
        _wrote(out)
    return (o, final, work) if keep else (o, final)


def delta_rule_backward(d_o, q, k, v, g, beta, scale=None, initial_state=None, offsets=None, d_final_state=None, saved=None):
    """Gradients of delta_rule: d_o [tokens, heads_v, width_v] of v's type and d_final_state float32 (default zero) in,
    -> (dq, dk, dv, dg, dbeta, d_initial_state); dq and dk are summed over the value heads that share a head.  The other
    arguments are those of the forward call; `saved` is what it returned with keep=True (without it the states are computed
    again).  d_initial_state is returned whether or not there was an initial state.  The results record no gradients of their own."""
    call = _Call(q, k, v, g, beta, scale, initial_state, offsets)
    _same_gpu("d_o", d_o, call.device)
    if d_o.dtype != call.dtype or tuple(d_o.shape) != (call.tokens, call.hv, call.dv):
        _fail("d_o must be %s %s" % (call.dtype, (call.tokens, call.hv, call.dv)))
    d_o = _inner(d_o, 16)
    d_final = _state("d_final_state", d_final_state, call.state_shape, call.device)
    _, kept, own = call.work
    if saved is None:
        _, saved = call.forward(None, True)
    else:
        _same_gpu("saved", saved, call.device)
        if saved.dtype != torch.uint8 or saved.numel() != kept or not saved.is_contiguous():
            _fail("saved is not what delta_rule(..., keep=True) returned for these arguments")
    dq, dk, dv, dg, dbeta = _like(q), _like(k), _like(v), _like(g), _like(beta)
    d_initial = q.new_empty(call.state_shape, dtype=torch.float32)
    work = q.new_empty(own, dtype=torch.uint8)
    op = call.pack(d_o=d_o, d_final=d_final, grads=(dq, dk, dv, dg, dbeta, d_initial))
    rc = _lib.load().helen_delta_rule_backward(op, saved.data_ptr(), kept, work.data_ptr(), own, _stream(call.device))
    if rc:
        _lib.check(rc)
    return dq, dk, dv, dg, dbeta, d_initial


def delta_rule_step(q, k, v, g, beta, state, slots=None, scale=None, out=None):
    """The same rule for one token per row over a pool of states, in place: q, k [rows, heads_k, width_k], v [rows, heads_v,
    width_v], g, beta [rows, heads_v], state float32 [pool, heads_v, width_k, width_v] (entries contiguous).
      slots   int32 [rows] on the GPU: the entry of each row (default: row i is entry i), some thousand of them at most (finding
              equal ones takes time with the square of the rows).  -1 is a padded row: its output is zero.  Rows that name the
              same entry are successive tokens of one stream, taken in the order of the rows.  Any other number outside the pool
              makes that row's output NaN and changes no state
    -> o [rows, heads_v, width_v]."""
    if _recorded(q, k, v, g, beta, state, out):
        _outside("delta_rule_step", "call it", state, out)
    device, code, n, hk, hv, dk, dv = _heads(q, k, v, g, beta)
    _same_gpu("state", state, device)
    s_shape = state.shape
    if state.dtype != torch.float32 or len(s_shape) != 4 or s_shape[1:] != (hv, dk, dv):
        _fail("state must be float32 [pool, %d, %d, %d]" % (hv, dk, dv))
    pool, per = s_shape[0], hv * dk * dv
    stride = per
    if pool > 0 and state.numel():
        strides = state.stride()
        if strides[1:] != (dk * dv, dv, 1) and not state[0].is_contiguous():
            _fail("the entries of state must be contiguous")
        stride = strides[0] if pool > 1 else per
        if stride < per or stride % 4 or state.data_ptr() % 16:
            _fail("the entries of state overlap or are not 16-byte aligned")
    if slots is None:
        if n > pool:
            _fail("%d rows over a pool of %d states" % (n, pool))
    else:
        _same_gpu("slots", slots, device)
        if slots.dtype != torch.int32 or slots.shape != (n,):
            _fail("slots must be int32 [%d]" % n)
        slots = slots.contiguous()
    if out is None:
        o = _like(v)
    else:
        o = _output("out", out, (n, hv, dv), q.dtype, device)
    q, k, v = _inner(q), _inner(k), _inner(v, 16)
    qs, ks, vs, gs, bs, os = q.stride(), k.stride(), v.stride(), g.stride(), beta.stride(), o.stride()
    op = _STEP.pack(_STEP.size, device, code, hk, hv, dk, dv, n, pool, dk ** -0.5 if scale is None else float(scale),
                    0 if slots is None else slots.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                    beta.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], gs[0], gs[1], bs[0], bs[1],
                    state.data_ptr(), stride, o.data_ptr(), os[0], os[1])
    rc = _lib.load().helen_delta_rule_step(op, _stream(device))
    if rc:
        _lib.check(rc)
    _wrote(state)
    if out is not None:
        _wrote(out)
    return o


def _rows(t):
    """`t` [..., width] as rows of one stride (a copy where its strides have no such form)."""
    t = _inner(t)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return _inner(t)


def _norm_sizes(x, weight, bias):
    """-> (device, type of x, type of the weight, width)."""
    device = _gpu_index("x", x)
    dtype = x.dtype
    code = _TYPES.get(dtype)
    if code is None:
        _fail("x is %s: float32, bfloat16 or float16 are supported" % dtype)
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        _fail("x must have a last dimension of at least one element")
    width = shape[-1]
    kind = None
    for label, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _same_gpu(label, t, device)
            if t.shape != (width,):
                _fail("%s must be [%d]" % (label, width))
            of = t.dtype
            if of != dtype and of != torch.float32:
                _fail("%s is %s: x's type %s or float32 is needed" % (label, of, dtype))
            if kind is not None and kind != of:
                _fail("weight and bias must be of one type")
            kind = of
    return device, code, _lib.HELEN_TYPE_FP32 if kind is None else _TYPES[kind], width


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """Layer norm over the last dimension: y = (x - mean) rstd weight + bias with rstd = 1 / sqrt(var + eps).
    x [..., width] float32, bfloat16 or float16, weight / bias [width] of x's type or float32.  Rows of any stride and
    alignment, less than 2^24 of them in one call where they are longer than 16 KiB; `out` may be x itself.
    -> (y, mean, rstd), mean and rstd float32 [...] for layer_norm_backward."""
    if _recorded(x, weight, bias, out):
        _outside("layer_norm", "use LayerNorm.apply, or call it", out)
    device, code, kind, width = _norm_sizes(x, weight, bias)
    rows = _rows(x)
    shape = x.shape
    if out is None:
        y = _like(x)
    else:
        y = _output("out", out, tuple(shape), x.dtype, device)
        if y.dim() != 2 and not y.is_contiguous():
            _fail("out must be contiguous or have two dimensions")
    flat = y if y.dim() == 2 else y.view(-1, width)
    mean = x.new_empty(shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    op = _NORM.pack(_NORM.size, device, code, kind, width, rows.shape[0], eps, rows.data_ptr(), rows.stride(0), _ptr(weight),
                    _ptr(bias), flat.data_ptr(), flat.stride(0), mean.data_ptr(), rstd.data_ptr(), 0, 0, 0, 0, 0, 0)
    rc = _lib.load().helen_layer_norm_forward(op, _stream(device))
    if rc:
        _lib.check(rc)
    if out is not None:
        _wrote(out)
    return y, mean, rstd


@functools.lru_cache(maxsize=1024)
def _norm_bytes(code, kind, width, rows):
    op = _NORM.pack(_NORM.size, 0, code, kind, width, rows, 0.0, *(0,) * 14)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().helen_layer_norm_bytes(op, ctypes.byref(need)))
    return int(need.value)


def layer_norm_backward(dy, x, weight, mean, rstd, bias=True):
    """Gradients of layer_norm: dy like x, weight (or None), mean and rstd as layer_norm returned them
    -> (dx, dweight, dbias); dweight is None without a weight, dbias None with bias=False.  dweight and dbias have the weight's
    type (float32 without one) and are summed in float32 in a fixed order.  The results record no gradients of their own."""
    device, code, kind, width = _norm_sizes(x, weight, None)
    shape = x.shape
    _same_gpu("dy", dy, device)
    if dy.dtype != x.dtype or dy.shape != shape:
        _fail("dy must be %s %s" % (x.dtype, tuple(shape)))
    for name, t in (("mean", mean), ("rstd", rstd)):
        _same_gpu(name, t, device)
        if t.dtype != torch.float32 or t.shape != shape[:-1]:
            _fail("%s must be float32 %s" % (name, tuple(shape[:-1])))
    rows, drows = _rows(x), _rows(dy)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    weight = None if weight is None else weight.contiguous()
    dx = _like(x)
    flat = dx if dx.dim() == 2 else dx.view(-1, width)
    dweight = None if weight is None else torch.empty_like(weight)
    dbias = None
    if bias:
        dbias = x.new_empty(width, dtype=torch.float32) if weight is None else torch.empty_like(weight)
    n = rows.shape[0]
    size = _norm_bytes(code, kind, width, n)
    work = x.new_empty(size, dtype=torch.uint8)
    op = _NORM.pack(_NORM.size, device, code, kind, width, n, 0.0, rows.data_ptr(), rows.stride(0), _ptr(weight), 0, 0, 0,
                    mean.data_ptr(), rstd.data_ptr(), drows.data_ptr(), drows.stride(0), flat.data_ptr(), flat.stride(0),
                    _ptr(dweight), _ptr(dbias))
    rc = _lib.load().helen_layer_norm_backward(op, work.data_ptr(), size, _stream(device))
    if rc:
        _lib.check(rc)
    return dx, dweight, dbias


def _no_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("%s under autograd cannot be captured into a graph: torch would add into gradients of leaves that "
                           "belong to other streams; capture the explicit forward and backward calls instead" % what)


class DeltaRule(torch.autograd.Function):
    """delta_rule under autograd: DeltaRule.apply(q, k, v, g, beta, scale, initial_state, offsets) -> (o, final_state).
    Keeps what delta_rule(keep=True) returns for the backward pass where gradients are recorded (torch.utils.checkpoint around it, or
    delta_rule_backward without `saved`, computes it again instead); neither pass may be captured then (the explicit calls may).
    Otherwise it is the plain call."""

    @classmethod
    def apply(cls, q, k, v, g, beta, scale=None, initial_state=None, offsets=None):
        if _recorded(q, k, v, g, beta, initial_state):
            return super().apply(q, k, v, g, beta, scale, initial_state, offsets)
        return delta_rule(q, k, v, g, beta, scale, initial_state, offsets)

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale=None, initial_state=None, offsets=None):
        _no_capture("DeltaRule")
        o, final, saved = delta_rule(q, k, v, g, beta, scale, initial_state, offsets, keep=True)
        if isinstance(offsets, (list, tuple)):
            offsets = torch.tensor(offsets, dtype=torch.int64)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, g, beta, initial_state, offsets, saved)
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_final):
        _no_capture("DeltaRule")
        q, k, v, g, beta, initial, offsets, saved = ctx.saved_tensors
        dq, dk, dv, dg, dbeta, d0 = delta_rule_backward(d_o, q, k, v, g, beta, ctx.scale, initial, offsets, d_final, saved)
        return dq, dk, dv, dg, dbeta, None, d0 if initial is not None else None, None


class LayerNorm(torch.autograd.Function):
    """layer_norm under autograd: LayerNorm.apply(x, weight, bias, eps) -> y.  Where gradients are recorded neither pass may be
    captured (the explicit calls may); otherwise it is the plain call."""

    @classmethod
    def apply(cls, x, weight=None, bias=None, eps=1e-5):
        if _recorded(x, weight, bias):
            return super().apply(x, weight, bias, eps)
        return layer_norm(x, weight, bias, eps)[0]

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        _no_capture("LayerNorm")
        y, mean, rstd = layer_norm(x, weight, bias, eps)
        ctx.with_bias = bias is not None
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_capture("LayerNorm")
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dweight, dbias = layer_norm_backward(dy, x, weight, mean, rstd, bias=ctx.with_bias)
        return dx, dweight, None if dbias is None else dbias.to(ctx.bias_dtype), None
