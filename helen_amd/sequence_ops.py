"""Sequence operators on the MI355X: the gated delta rule (whole sequences, forward and backward, and single tokens over a
pool of states) and layer norm (forward and backward).

They stand beside HelenEngine.chunk_forward, the GRU layer with a carried hidden state: torch tensors in, torch tensors out,
all compute in libhelen_hip.so (include/helen_hip.h), asynchronous on the current stream of the tensors' device.  Gradients
are calls of their own; `DeltaRule` and `LayerNorm` tie them into torch's autograd.

A call keeps nothing: workspaces come from torch's allocator, so calls on several streams may run at once and a call may be
captured into a graph.  Nothing here waits for the device.
"""
import ctypes

import torch

from . import _lib

_TYPES = {torch.float32: _lib.HELEN_TYPE_FP32, torch.bfloat16: _lib.HELEN_TYPE_BF16, torch.float16: _lib.HELEN_TYPE_FP16}


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _on_gpu(name, t, device=None):
    _need(isinstance(t, torch.Tensor), "%s must be a torch tensor" % name)
    if not t.is_cuda:
        raise RuntimeError("%s is not on a GPU: the sequence operators need one, there is no CPU fallback" % name)
    _need(device is None or t.device == device, "%s is on %s, the other tensors on %s" % (name, t.device, device))


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _inner(t, bytes_=0):
    """`t` with a contiguous last dimension and, where `bytes_` is given, base and strides that are multiples of it; a copy if
    it has to be one."""
    if t.numel() and t.stride(-1) != 1 and t.shape[-1] != 1:
        return t.contiguous()
    if bytes_ and (t.data_ptr() % bytes_ or any(s * t.element_size() % bytes_ for s in t.stride()[:-1]) or t.stride(0) > 1 << 24):
        return t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else t.contiguous()
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _pair(t):
    return (ctypes.c_int64 * 2)(t.stride(0), t.stride(1))


def _heads(q, k, v, g, beta):
    """Types, devices and shapes of a call's tokens: -> (tokens, heads_k, heads_v, width_k, width_v)."""
    _on_gpu("q", q)
    for name, t in (("k", k), ("v", v), ("g", g), ("beta", beta)):
        _on_gpu(name, t, q.device)
    _need(q.dtype in _TYPES, "q is %s: float32, bfloat16 or float16 are supported" % q.dtype)
    _need(k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v are %s, %s, %s: one type is needed" % (q.dtype, k.dtype, v.dtype))
    _need(g.dtype == torch.float32 and beta.dtype == torch.float32, "g and beta must be float32")
    _need(q.dim() == 3 and v.dim() == 3, "q, k, v must be [tokens, heads, width]")
    _need(k.shape == q.shape, "k is %s, q %s" % (tuple(k.shape), tuple(q.shape)))
    n, hk, dk = q.shape
    hv, dv = v.shape[1:]
    _need(v.shape[0] == n, "v has %d tokens, q %d" % (v.shape[0], n))
    _need(tuple(g.shape) == (n, hv) and tuple(beta.shape) == (n, hv),
          "g and beta must be [%d, %d]: they are %s and %s" % (n, hv, tuple(g.shape), tuple(beta.shape)))
    _need(dk in (64, 128), "width %d of q and k: 64 and 128 are supported" % dk)
    _need(dv in (64, 128, 192, 256), "width %d of v: 64, 128, 192 and 256 are supported" % dv)
    _need(hk > 0 and hv > 0 and hv % hk == 0, "%d value heads do not share %d key heads evenly" % (hv, hk))
    _need(n < 2 ** 31, "%d tokens in one call" % n)
    return n, hk, hv, dk, dv


def _state(name, t, shape, device):
    if t is None:
        return None
    _on_gpu(name, t, device)
    _need(t.dtype == torch.float32 and tuple(t.shape) == shape, "%s must be float32 %s" % (name, shape))
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _output(name, t, shape, dtype, device):
    _on_gpu(name, t, device)
    _need(t.dtype == dtype and tuple(t.shape) == shape, "%s must be %s %s" % (name, dtype, shape))
    _need(t.numel() == 0 or t.stride(-1) == 1, "%s must have a contiguous last dimension" % name)
    return t


class _Call(object):
    """A checked delta rule call: the C description and the tensors it points into."""

    def __init__(self, q, k, v, g, beta, scale, initial_state, offsets):
        self.tokens, self.hk, self.hv, self.dk, self.dv = _heads(q, k, v, g, beta)
        self.device, self.dtype = q.device, q.dtype
        self.q, self.k, self.v = _inner(q, 16), _inner(k, 16), _inner(v, 16)
        self.g, self.beta = g, beta
        whole = True                       # every row belongs to a sequence, as far as the host can tell
        if offsets is None:
            sequences = 1
            self.offsets = None
        else:
            if isinstance(offsets, (list, tuple)):
                offsets = torch.tensor(offsets, dtype=torch.int64)
            _need(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.numel() >= 2
                  and offsets.dtype in (torch.int32, torch.int64), "offsets must be one row of at least two int32 / int64")
            sequences = offsets.numel() - 1
            whole = False
            if offsets.is_cuda:
                _on_gpu("offsets", offsets, q.device)
            else:
                at = offsets.tolist()
                _need(at[0] == 0 and at[-1] <= self.tokens and all(a <= b for a, b in zip(at, at[1:])),
                      "offsets must ascend from 0 to at most %d" % self.tokens)
                whole = at[-1] == self.tokens
            self.offsets = offsets.to(device=q.device, dtype=torch.int32).contiguous()
        self.sequences = sequences
        self.whole = whole
        self.state_shape = (sequences, self.hv, self.dk, self.dv)
        self.initial = _state("initial_state", initial_state, self.state_shape, q.device)
        c = self.c = _lib.HelenDeltaRuleC()
        c.struct_size = ctypes.sizeof(c)
        c.device, c.dtype = q.device.index, _TYPES[q.dtype]
        c.heads_k, c.heads_v, c.width_k, c.width_v = self.hk, self.hv, self.dk, self.dv
        c.tokens, c.sequences = self.tokens, sequences
        c.scale = float(self.dk ** -0.5 if scale is None else scale)
        c.offsets = _ptr(self.offsets)
        c.q, c.k, c.v, c.g, c.beta = (_ptr(t) for t in (self.q, self.k, self.v, self.g, self.beta))
        c.q_stride, c.k_stride, c.v_stride = _pair(self.q), _pair(self.k), _pair(self.v)
        c.g_stride, c.beta_stride = _pair(self.g), _pair(self.beta)
        c.initial_state = _ptr(self.initial)

    def bytes(self):
        got = [ctypes.c_size_t() for _ in range(3)]
        _lib.check(_lib.load().helen_delta_rule_bytes(ctypes.byref(self.c), *(ctypes.byref(x) for x in got)))
        return [int(x.value) for x in got]

    def forward(self, o, keep):
        """-> (final_state, workspace); `o` None computes the states alone."""
        final = torch.empty(self.state_shape, dtype=torch.float32, device=self.device)
        c = self.c
        c.o, c.final_state = _ptr(o), final.data_ptr()
        if o is not None:
            c.o_stride = _pair(o)
        plain, kept, _ = self.bytes()
        work = torch.empty(kept if keep else plain, dtype=torch.uint8, device=self.device)
        _lib.check(_lib.load().helen_delta_rule_forward(ctypes.byref(c), int(keep), work.data_ptr(), work.numel(),
                                                        _stream(self.device)))
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
      keep           True: also return what delta_rule_backward needs of this call
    -> (o, final_state) or (o, final_state, saved).  States stay float32-class whatever the type of q, k, v."""
    call = _Call(q, k, v, g, beta, scale, initial_state, offsets)
    shape = (call.tokens, call.hv, call.dv)
    if out is None:
        o = torch.empty(shape, dtype=call.dtype, device=call.device)
        call.c.zero_tail = 0 if call.whole else 1
    else:
        o = _output("out", out, shape, call.dtype, call.device)
    final, work = call.forward(o, keep)
    return (o, final, work) if keep else (o, final)


def delta_rule_backward(d_o, q, k, v, g, beta, scale=None, initial_state=None, offsets=None, d_final_state=None, saved=None):
    """Gradients of delta_rule: d_o [tokens, heads_v, width_v] of v's type and d_final_state float32 (default zero) in,
    -> (dq, dk, dv, dg, dbeta, d_initial_state); dq and dk are summed over the value heads that share a head.  The other
    arguments are those of the forward call; `saved` is what it returned with keep=True (without it the states are computed
    again).  d_initial_state is returned whether or not there was an initial state."""
    call = _Call(q, k, v, g, beta, scale, initial_state, offsets)
    _on_gpu("d_o", d_o, call.device)
    _need(d_o.dtype == call.dtype and tuple(d_o.shape) == (call.tokens, call.hv, call.dv),
          "d_o must be %s %s" % (call.dtype, (call.tokens, call.hv, call.dv)))
    d_o = _inner(d_o, 16)
    d_final = _state("d_final_state", d_final_state, call.state_shape, call.device)
    _, kept, own = call.bytes()
    if saved is None:
        _, saved = call.forward(None, True)
    else:
        _on_gpu("saved", saved, call.device)
        _need(saved.dtype == torch.uint8 and saved.numel() == kept and saved.is_contiguous(),
              "saved is not what delta_rule(..., keep=True) returned for these arguments")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    dg, dbeta = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (g, beta))
    d_initial = torch.empty(call.state_shape, dtype=torch.float32, device=call.device)
    c = call.c
    c.d_o, c.d_o_stride, c.d_final_state = d_o.data_ptr(), _pair(d_o), _ptr(d_final)
    c.grad_q, c.grad_k, c.grad_v, c.grad_g, c.grad_beta = (t.data_ptr() for t in (dq, dk, dv, dg, dbeta))
    c.grad_initial_state = d_initial.data_ptr()
    work = torch.empty(own, dtype=torch.uint8, device=call.device)
    _lib.check(_lib.load().helen_delta_rule_backward(ctypes.byref(c), saved.data_ptr(), saved.numel(), work.data_ptr(),
                                                     work.numel(), _stream(call.device)))
    return dq, dk, dv, dg, dbeta, d_initial


def delta_rule_step(q, k, v, g, beta, state, slots=None, scale=None, out=None):
    """The same rule for one token per row over a pool of states, in place: q, k [rows, heads_k, width_k], v [rows, heads_v,
    width_v], g, beta [rows, heads_v], state float32 [pool, heads_v, width_k, width_v] (entries contiguous).
      slots   int32 [rows] on the GPU: the entry of each row (default: row i is entry i).  -1 is a padded row: its output is
              zero.  Rows that name the same entry are successive tokens of one stream, taken in the order of the rows.  Any
              other number outside the pool makes that row's output NaN and changes no state
    -> o [rows, heads_v, width_v]."""
    n, hk, hv, dk, dv = _heads(q, k, v, g, beta)
    device = q.device
    _on_gpu("state", state, device)
    _need(state.dtype == torch.float32 and state.dim() == 4 and tuple(state.shape[1:]) == (hv, dk, dv),
          "state must be float32 [pool, %d, %d, %d]" % (hv, dk, dv))
    pool = state.shape[0]
    _need(pool == 0 or state[0].is_contiguous(), "the entries of state must be contiguous")
    per = hv * dk * dv
    stride = state.stride(0) if pool > 1 else per
    _need(stride >= per and stride % 4 == 0 and state.data_ptr() % 16 == 0, "the entries of state overlap or are not 16-byte aligned")
    if slots is None:
        _need(n <= pool, "%d rows over a pool of %d states" % (n, pool))
    else:
        _on_gpu("slots", slots, device)
        _need(slots.dtype == torch.int32 and tuple(slots.shape) == (n,), "slots must be int32 [%d]" % n)
        slots = slots.contiguous()
    if out is None:
        o = torch.empty((n, hv, dv), dtype=q.dtype, device=device)
    else:
        o = _output("out", out, (n, hv, dv), q.dtype, device)
    q, k, v = _inner(q), _inner(k), _inner(v, 16)
    c = _lib.HelenDeltaStepC()
    c.struct_size = ctypes.sizeof(c)
    c.device, c.dtype = device.index, _TYPES[q.dtype]
    c.heads_k, c.heads_v, c.width_k, c.width_v, c.rows, c.pool = hk, hv, dk, dv, n, pool
    c.scale = float(dk ** -0.5 if scale is None else scale)
    c.slots = _ptr(slots)
    c.q, c.k, c.v, c.g, c.beta, c.state, c.o = (t.data_ptr() for t in (q, k, v, g, beta, state, o))
    c.q_stride, c.k_stride, c.v_stride = _pair(q), _pair(k), _pair(v)
    c.g_stride, c.beta_stride, c.o_stride = _pair(g), _pair(beta), _pair(o)
    c.state_stride = stride
    _lib.check(_lib.load().helen_delta_rule_step(ctypes.byref(c), _stream(device)))
    return o


def _rows(t):
    """`t` [..., width] as rows of one stride (a copy where its strides have no such form)."""
    t = _inner(t)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return _inner(t)


def _norm_call(x, weight, bias, name):
    _on_gpu("x", x)
    _need(x.dtype in _TYPES, "x is %s: float32, bfloat16 or float16 are supported" % x.dtype)
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "x must have a last dimension of at least one element")
    width = x.shape[-1]
    kind = None
    for label, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _on_gpu(label, t, x.device)
            _need(tuple(t.shape) == (width,), "%s must be [%d]" % (label, width))
            _need(t.dtype in (x.dtype, torch.float32), "%s is %s: x's type %s or float32 is needed" % (label, t.dtype, x.dtype))
            _need(kind in (None, t.dtype), "weight and bias must be of one type")
            kind = t.dtype
    c = _lib.HelenLayerNormC()
    c.struct_size = ctypes.sizeof(c)
    c.device, c.dtype, c.weight_dtype = x.device.index, _TYPES[x.dtype], _TYPES[kind or torch.float32]
    c.width = width
    return c, width


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """Layer norm over the last dimension: y = (x - mean) rstd weight + bias with rstd = 1 / sqrt(var + eps).
    x [..., width] float32, bfloat16 or float16, weight / bias [width] of x's type or float32.  Rows of any stride and alignment.
    -> (y, mean, rstd), mean and rstd float32 [...] for layer_norm_backward."""
    c, width = _norm_call(x, weight, bias, "layer_norm")
    rows = _rows(x)
    n = rows.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else _output("out", out, tuple(x.shape), x.dtype, x.device)
    _need(out is None or y.is_contiguous() or y.dim() == 2, "out must be contiguous or have two dimensions")
    flat = y if y.dim() == 2 else y.view(-1, width)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    c.rows, c.eps = n, float(eps)
    c.x, c.x_stride, c.y, c.y_stride = rows.data_ptr(), rows.stride(0), flat.data_ptr(), flat.stride(0)
    c.weight, c.bias, c.mean, c.rstd = _ptr(weight), _ptr(bias), mean.data_ptr(), rstd.data_ptr()
    _lib.check(_lib.load().helen_layer_norm_forward(ctypes.byref(c), _stream(x.device)))
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, bias=True):
    """Gradients of layer_norm: dy like x, weight (or None), mean and rstd as layer_norm returned them
    -> (dx, dweight, dbias); dweight is None without a weight, dbias None with bias=False.  dweight and dbias have the weight's
    type (float32 without one) and are summed in float32 in a fixed order."""
    c, width = _norm_call(x, weight, None, "layer_norm_backward")
    _on_gpu("dy", dy, x.device)
    _need(dy.dtype == x.dtype and dy.shape == x.shape, "dy must be %s %s" % (x.dtype, tuple(x.shape)))
    for name, t in (("mean", mean), ("rstd", rstd)):
        _on_gpu(name, t, x.device)
        _need(t.dtype == torch.float32 and t.shape == x.shape[:-1], "%s must be float32 %s" % (name, tuple(x.shape[:-1])))
    rows, drows = _rows(x), _rows(dy)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    weight = None if weight is None else weight.contiguous()
    kind = torch.float32 if weight is None else weight.dtype
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    flat = dx if dx.dim() == 2 else dx.view(-1, width)
    dweight = None if weight is None else torch.empty(width, dtype=kind, device=x.device)
    dbias = torch.empty(width, dtype=kind, device=x.device) if bias else None
    c.rows = rows.shape[0]
    c.x, c.x_stride, c.dy, c.dy_stride = rows.data_ptr(), rows.stride(0), drows.data_ptr(), drows.stride(0)
    c.dx, c.dx_stride = flat.data_ptr(), flat.stride(0)
    c.weight, c.mean, c.rstd, c.dweight, c.dbias = _ptr(weight), mean.data_ptr(), rstd.data_ptr(), _ptr(dweight), _ptr(dbias)
    lib = _lib.load()
    need = ctypes.c_size_t()
    _lib.check(lib.helen_layer_norm_bytes(ctypes.byref(c), ctypes.byref(need)))
    work = torch.empty(max(int(need.value), 16), dtype=torch.uint8, device=x.device)
    _lib.check(lib.helen_layer_norm_backward(ctypes.byref(c), work.data_ptr(), work.numel(), _stream(x.device)))
    return dx, dweight, dbias


def _no_capture(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("%s under autograd cannot be captured into a graph: torch would add into gradients of leaves that "
                           "belong to other streams; capture the explicit forward and backward calls instead" % what)


class DeltaRule(torch.autograd.Function):
    """delta_rule under autograd: DeltaRule.apply(q, k, v, g, beta, scale, initial_state, offsets) -> (o, final_state).
    Keeps the forward call's states for the backward pass.  Not capturable: the explicit calls are."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale=None, initial_state=None, offsets=None):
        _no_capture("DeltaRule")
        keep = any(ctx.needs_input_grad)
        got = delta_rule(q, k, v, g, beta, scale, initial_state, offsets, keep=keep)
        if keep:
            if isinstance(offsets, (list, tuple)):
                offsets = torch.tensor(offsets, dtype=torch.int64)
            ctx.scale = scale
            ctx.save_for_backward(q, k, v, g, beta, initial_state, offsets, got[2])
        return got[0], got[1]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_final):
        _no_capture("DeltaRule")
        q, k, v, g, beta, initial, offsets, saved = ctx.saved_tensors
        dq, dk, dv, dg, dbeta, d0 = delta_rule_backward(d_o, q, k, v, g, beta, ctx.scale, initial, offsets, d_final, saved)
        return dq, dk, dv, dg, dbeta, None, d0 if initial is not None else None, None


class LayerNorm(torch.autograd.Function):
    """layer_norm under autograd: LayerNorm.apply(x, weight, bias, eps) -> y.  Not capturable: the explicit calls are."""

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
