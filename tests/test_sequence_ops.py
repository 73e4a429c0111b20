"""The sequence operators (helen_amd.sequence_ops): the gated delta rule forward, backward and single-token, and layer norm
forward and backward, against their definitions in 64 bits.

Tolerances, with u = 2^-24 and half = eps / 2 of the output's type (one rounding of the result).  The operators compute in
fp32-class arithmetic: a sum of n products is off by at most n u of the sum of magnitudes, and by about sqrt(n) u of its own
size when the errors are independent, which is what the 2-norms below see.
  delta rule: a result goes through at most 8 such sums of n <= width_k + width_v + 64 products, one after another.  In the
    2-norm 8 sqrt(n) u (n = 320: 8.5e-6), in a single element 8 n u of the largest result.  A state handed on through a chain
    does not add to that: beta k k^T with |k| = 1, beta <= 1 and e^g <= 1 never lengthens an error, and a chain here has at most
    6 chunks: factor 6 on the single element's bound, sqrt(6) on the norm's.
    Outputs of 16 bits take P U with two terms an operand, 2^-16 of each: at most 2 2^-16 of the sum of magnitudes.
  layer norm: 3 sums of `width` terms (in pieces: n u at worst, sqrt(n) u in the norm), dweight and dbias one of `rows` terms."""
import ctypes
import math

import pytest
import torch

from helen_amd import _lib, sequence_ops as ops

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------------------------------------------------ references
def delta_reference(q, k, v, g, beta, scale, initial, lengths):
    """Token by token in float64 on the CPU, differentiable."""
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    outs, states, at = [], [], 0
    for i, n in enumerate(lengths):
        S = initial[i] if initial is not None else q.new_zeros(v.shape[1], q.shape[2], v.shape[2])
        for t in range(at, at + n):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (k[t][:, None, :] @ S)[:, 0])
            S = S + k[t][:, :, None] * u[:, None, :]
            outs.append(scale * (q[t][:, None, :] @ S)[:, 0])
        states.append(S)
        at += n
    return (torch.stack(outs) if outs else v[:0] * 1.0), torch.stack(states)


def make(lengths, hk, hv, dk, dv, dtype, initial, seed=0, tail=0, decay=1.0):
    gen = torch.Generator().manual_seed(seed)
    n = sum(lengths) + tail
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    return dict(q=unit(rand(n, hk, dk)).to(dtype), k=unit(rand(n, hk, dk)).to(dtype), v=rand(n, hv, dv).to(dtype),
                g=-decay * rand(n, hv).abs() * torch.linspace(0.02, 2.0, hv), beta=torch.sigmoid(rand(n, hv)),
                initial=0.3 * rand(len(lengths), hv, dk, dv) if initial else None,
                do=rand(n, hv, dv).to(dtype), ds=0.3 * rand(len(lengths), hv, dk, dv) if initial else None,
                scale=dk ** -0.5)


def gpu(x):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in x.items()}


def ends(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def close(name, got, want, n, chunks=1, two_terms=False):
    got = got.detach().cpu()
    t = got.dtype
    round_ = half(t) if t != torch.float32 else U
    got = got.double()
    want = want.detach()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if not want.numel():
        return
    top = float(want.abs().max())
    arith = 8 * n * chunks * U + (2 * 2.0 ** -16 if two_terms else 0.0)
    off = (got - want).abs()
    bound = round_ * want.abs() + arith * top + 1e-30
    assert bool((off <= bound).all()), "%s: off by %.3g where %.3g is allowed" % (name, float((off - bound).max()), float(bound.max()))
    norm = float(off.norm() / want.norm()) if float(want.norm()) else float(off.norm())
    allowed = round_ + 8 * math.sqrt(n * chunks) * U + (2 * 2.0 ** -16 if two_terms else 0.0)
    assert norm <= allowed, "%s: %.3g of the norm, %.3g allowed" % (name, norm, allowed)


def check_delta(x, lengths, backward=True, offsets="gpu"):
    d = gpu(x)
    live = sum(lengths)
    off = ends(lengths)
    if offsets == "gpu":
        off = torch.tensor(off, dtype=torch.int32).cuda()
    elif offsets is None:
        assert len(lengths) == 1
    args = (d["q"], d["k"], d["v"], d["g"], d["beta"])
    kw = dict(scale=x["scale"], initial_state=d["initial"], offsets=off if offsets else None)
    o, s, saved = ops.delta_rule(*args, keep=True, **kw)
    o2, s2 = ops.delta_rule(*args, **kw)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    leaves = [x[n].double()[:live].requires_grad_() for n in ("q", "k", "v", "g", "beta")]
    first = x["initial"].double().requires_grad_() if x["initial"] is not None else None
    ro, rs = delta_reference(*leaves, x["scale"], first, lengths)
    n = x["q"].shape[2] + x["v"].shape[2] + 64
    chunks = max(1, max((m + 63) // 64 for m in lengths))
    sixteen = x["q"].dtype != torch.float32
    close("o", o[:live], ro, n, chunks, sixteen)
    close("final_state", s, rs, n, chunks)
    assert not o[live:].any()
    if not backward:
        return
    got = ops.delta_rule_backward(d["do"], *args, d_final_state=d["ds"], saved=saved, **kw)
    again = ops.delta_rule_backward(d["do"], *args, d_final_state=d["ds"], **kw)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    loss = (ro * x["do"].double()[:live]).sum()
    if x["ds"] is not None:
        loss = loss + (rs * x["ds"].double()).sum()
    wanted = torch.autograd.grad(loss, leaves + ([first] if first is not None else []), allow_unused=True)
    names = ("dq", "dk", "dv", "dg", "dbeta", "d_initial")
    for name, a, b in zip(names, got, wanted):
        if b is None:
            b = torch.zeros(a.shape if name == "d_initial" else (live,) + a.shape[1:], dtype=torch.float64)
        if name != "d_initial":
            assert not a[live:].any(), name
            a = a[:live]
        close(name, a, b, n, chunks)


# ------------------------------------------------------------------------------------------------------------- refusals
def description(**change):
    c = _lib.HelenDeltaRuleC()
    c.struct_size = ctypes.sizeof(c)
    c.dtype, c.heads_k, c.heads_v, c.width_k, c.width_v, c.tokens, c.sequences = 1, 2, 4, 128, 128, 100, 1
    for k, v in change.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("change, text", [
    (dict(struct_size=8), b"struct_size"), (dict(dtype=3), b"dtype"), (dict(width_k=96), b"width_k"),
    (dict(width_v=32), b"width_v"), (dict(width_v=320), b"width_v"), (dict(heads_v=3), b"share"), (dict(heads_k=0), b"share"),
    (dict(tokens=-1), b"tokens"), (dict(sequences=0), b"sequences"), (dict(sequences=3), b"one length"),
    (dict(tokens=2 ** 31 - 1, heads_k=64, heads_v=64), b"more than one call"), (dict(), b"null input"),
])
def test_delta_rule_refuses(change, text):
    lib = _lib.load()
    assert lib.helen_delta_rule_forward(ctypes.byref(description(**change)), 0, None, 0, None) == -1
    assert text in lib.helen_last_error(), lib.helen_last_error()


def test_delta_rule_refuses_null_workspace_and_misaligned_inputs():
    lib = _lib.load()
    base = dict(q=4096, k=4096, v=4096, g=4096, beta=4096)
    even = (ctypes.c_int64 * 2)(512, 128)
    c = description(q_stride=even, k_stride=even, v_stride=even, **base)
    assert lib.helen_delta_rule_forward(ctypes.byref(c), 0, None, 0, None) == -1 and b"workspace" in lib.helen_last_error()
    assert lib.helen_delta_rule_backward(ctypes.byref(c), None, 0, None, 0, None) == -1 and b"null gradient" in lib.helen_last_error()
    c.q = 4098
    assert lib.helen_delta_rule_forward(ctypes.byref(c), 0, None, 0, None) == -1 and b"16 bytes" in lib.helen_last_error()
    c.q, c.k_stride = 4096, (ctypes.c_int64 * 2)(515, 128)
    assert lib.helen_delta_rule_forward(ctypes.byref(c), 0, None, 0, None) == -1 and b"16 bytes" in lib.helen_last_error()
    assert lib.helen_delta_rule_bytes(None, None, None, None) == -1
    got = [ctypes.c_size_t() for _ in range(3)]
    assert lib.helen_delta_rule_bytes(ctypes.byref(description()), *(ctypes.byref(x) for x in got)) == 0
    assert 0 < got[0].value < got[1].value and got[2].value > 0


@pytest.mark.parametrize("change, text", [
    (dict(struct_size=8), b"struct_size"), (dict(dtype=9), b"dtype"), (dict(width_k=32), b"width_k"),
    (dict(width_v=100), b"width_v"), (dict(heads_v=5), b"share"), (dict(rows=-1), b"rows"), (dict(rows=9), b"pool"),
    (dict(), b"null"),
])
def test_delta_step_refuses(change, text):
    lib = _lib.load()
    c = _lib.HelenDeltaStepC()
    c.struct_size = ctypes.sizeof(c)
    c.heads_k, c.heads_v, c.width_k, c.width_v, c.rows, c.pool = 2, 4, 128, 128, 4, 8
    for k, v in change.items():
        setattr(c, k, v)
    assert lib.helen_delta_rule_step(ctypes.byref(c), None) == -1
    assert text in lib.helen_last_error(), lib.helen_last_error()


@pytest.mark.parametrize("change, text", [
    (dict(struct_size=8), b"struct_size"), (dict(dtype=5), b"dtype"), (dict(weight_dtype=2), b"weight"),
    (dict(width=0), b"width"), (dict(rows=-1), b"rows"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"),
    (dict(rows=2 ** 40), b"more than one call"), (dict(), b"null"),
])
def test_layer_norm_refuses(change, text):
    lib = _lib.load()
    c = _lib.HelenLayerNormC()
    c.struct_size = ctypes.sizeof(c)
    c.dtype, c.weight_dtype, c.width, c.rows, c.eps = 1, 1, 128, 4, 1e-5
    for k, v in change.items():
        setattr(c, k, v)
    assert lib.helen_layer_norm_forward(ctypes.byref(c), None) == -1
    assert text in lib.helen_last_error(), lib.helen_last_error()
    assert lib.helen_layer_norm_backward(ctypes.byref(c), None, 0, None) == -1


@pytest.mark.parametrize("packer, structure", [("_RULE", "HelenDeltaRuleC"), ("_STEP", "HelenDeltaStepC"), ("_NORM", "HelenLayerNormC")])
def test_packed_descriptions_have_the_layout_of_the_structures(packer, structure):
    packer, structure = getattr(ops, packer), getattr(_lib, structure)
    assert packer.size == ctypes.sizeof(structure)
    count = len(packer.unpack(bytes(packer.size)))
    got = structure.from_buffer_copy(packer.pack(*range(1, count + 1)))
    flat = []
    for name, _ in structure._fields_:
        value = getattr(got, name)
        flat += list(value) if hasattr(value, "__len__") else [value]
    assert [int(x) for x in flat] == list(range(1, count + 1))


def test_tensors_on_the_host_are_refused():
    x = make([4], 1, 1, 64, 64, torch.float32, False)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.delta_rule_step(x["q"], x["k"], x["v"], x["g"], x["beta"], torch.zeros(4, 1, 64, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.layer_norm(torch.zeros(2, 8))


@pytest.mark.gpu
def test_shapes_types_and_offsets_are_refused():
    x = gpu(make([10], 2, 4, 64, 64, torch.bfloat16, False))
    a = dict(q=x["q"], k=x["k"], v=x["v"], g=x["g"], beta=x["beta"])

    def refused(match, **change):
        with pytest.raises(ValueError, match=match):
            ops.delta_rule(**dict(a, **change))
    refused("one type", k=x["k"].float())
    refused("supported", q=x["q"].double(), k=x["k"].double(), v=x["v"].double())
    refused("float32", g=x["g"].half())
    refused("k is", k=x["k"][:, :, :32])
    refused("width 32", q=x["q"][:, :, :32], k=x["k"][:, :, :32])
    refused("width 32 of v", v=x["v"][:, :, :32])
    refused("tokens", v=x["v"][:9], g=x["g"][:9], beta=x["beta"][:9])
    refused("g and beta", beta=x["beta"][:, :2])
    refused("evenly", v=x["v"][:, :3], g=x["g"][:, :3], beta=x["beta"][:, :3])
    refused("ascend", offsets=[0, 11])
    refused("ascend", offsets=[1, 10])
    refused("ascend", offsets=[0, 7, 5, 10])
    refused("offsets", offsets=torch.zeros(1, dtype=torch.int32))
    refused("offsets", offsets=torch.zeros(2))
    refused("initial_state", initial_state=torch.zeros(2, 4, 64, 64, device="cuda"))
    refused("out", out=torch.zeros(10, 4, 64, device="cuda"))
    with pytest.raises(ValueError, match="d_o"):
        ops.delta_rule_backward(x["do"].float(), **a)
    with pytest.raises(ValueError, match="saved"):
        ops.delta_rule_backward(x["do"], saved=torch.zeros(64, dtype=torch.uint8, device="cuda"), **a)
    with pytest.raises(ValueError, match="rows over a pool"):
        ops.delta_rule_step(state=torch.zeros(9, 4, 64, 64, device="cuda"), **a)
    with pytest.raises(ValueError, match="slots"):
        ops.delta_rule_step(state=torch.zeros(9, 4, 64, 64, device="cuda"), slots=torch.zeros(10, device="cuda"), **a)
    with pytest.raises(ValueError, match="state"):
        ops.delta_rule_step(state=torch.zeros(10, 4, 64, 64, device="cuda").bfloat16(), **a)
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x["v"], torch.zeros(64, device="cuda").half())
    with pytest.raises(ValueError, match="dy"):
        ops.layer_norm_backward(x["v"].float(), x["v"], None, *ops.layer_norm(x["v"])[1:])


# ----------------------------------------------------------------------------------------------------------- delta rule
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("lengths", [[1], [63], [64], [65], [200]])
def test_delta_rule_one_sequence(dtype, lengths):
    check_delta(make(lengths, 1, 2, 128, 128, TYPES[dtype], lengths != [64], seed=lengths[0]), lengths, offsets=None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, hk, hv, dk, dv", [
    ("fp32", 1, 1, 64, 64), ("bf16", 2, 2, 64, 128), ("fp16", 1, 3, 64, 192), ("bf16", 2, 4, 128, 64),
    ("fp32", 1, 2, 128, 256), ("fp16", 3, 3, 128, 128),
])
def test_delta_rule_packed_sequences(dtype, hk, hv, dk, dv):
    lengths = [1, 0, 63, 64, 65, 0, 130, 5, 0]
    check_delta(make(lengths, hk, hv, dk, dv, TYPES[dtype], True, seed=7, tail=0), lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("hk, hv, dk, dv", [(4, 8, 128, 128), (16, 16, 64, 64), (5, 5, 128, 256)])
def test_delta_rule_more_chains_than_compute_units(dtype, hk, hv, dk, dv):
    """320 and 400 chains of 16 columns (the other tests' few sequences stay below 256)."""
    lengths = [70, 64, 1, 131, 33]
    check_delta(make(lengths, hk, hv, dk, dv, TYPES[dtype], True, seed=hv), lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dk", [64, 128])
def test_delta_rule_more_chains_with_strided_and_short_inputs(dk):
    """The chains that read q and k themselves: slices of one projection, heads first, broadcast keys, the last row the last of
    its allocation."""
    lengths = [70, 64, 1, 131, 33]
    n = sum(lengths)
    x = gpu(make(lengths, 4, 8, dk, 128, torch.bfloat16, True, seed=dk))
    off = torch.tensor(ends(lengths), dtype=torch.int32).cuda()
    kw = dict(initial_state=x["initial"], offsets=off)

    def run(q, k):
        return ops.delta_rule(q, k, x["v"], x["g"], x["beta"], **kw)
    want = run(x["q"], x["k"])
    kept = ops.delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], keep=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, kept))
    rows = torch.cat([x["q"].reshape(n, -1), x["k"].reshape(n, -1)], 1)
    first = {m: x[m].transpose(0, 1).contiguous().transpose(0, 1) for m in ("q", "k")}
    for q, k in ((rows[:, :4 * dk].unflatten(1, (4, dk)), rows[:, 4 * dk:].unflatten(1, (4, dk))), (first["q"], first["k"])):
        assert q.data_ptr() % 16 == 0 and not q.is_contiguous()
        assert all(torch.equal(a, b) for a, b in zip(run(q, k), want))
    one = x["k"][:1].expand(n, -1, -1)
    assert all(torch.equal(a, b) for a, b in zip(run(x["q"], one), run(x["q"], one.contiguous())))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("hk, hv, dk, dv", [(1, 2, 128, 128), (2, 2, 64, 256)])
def test_delta_rule_six_chunks(dtype, hk, hv, dk, dv):
    lengths = [380, 320]
    check_delta(make(lengths, hk, hv, dk, dv, TYPES[dtype], True, seed=dv), lengths)


@pytest.mark.gpu
def test_outputs_that_overlap_and_host_offsets_in_a_capture_are_refused():
    x = gpu(make([10], 1, 2, 64, 64, torch.float32, False))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    row = torch.zeros(1, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        ops.delta_rule(*args, out=row.expand(10, 2, 64))
    with pytest.raises(ValueError, match="overlap"):
        ops.delta_rule_step(*args, torch.zeros(10, 2, 64, 64, device="cuda"), out=torch.zeros(200, device="cuda").as_strided((10, 2, 64), (6, 64, 1)))
    with pytest.raises(ValueError, match="overlap"):
        ops.layer_norm(x["v"], out=row[:, :1].expand(10, 2, 64))
    want = ops.delta_rule(*args, offsets=torch.tensor([0, 3, 10], dtype=torch.int32, device="cuda"))
    apart = torch.zeros(2, 10, 64, device="cuda").transpose(0, 1)
    got = ops.delta_rule(*args, offsets=[0, 3, 10], out=apart)
    assert got[0].data_ptr() == apart.data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x["v"] * 2
        with pytest.raises(RuntimeError, match="host cannot be captured"):
            ops.delta_rule(*args, offsets=[0, 3, 10])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x["v"] * 2)


@pytest.mark.gpu
def test_delta_rule_many_short_sequences():
    lengths = [(7 * i) % 5 for i in range(300)]
    check_delta(make(lengths, 1, 1, 64, 64, torch.bfloat16, False, seed=3), lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [1, 64, 200])
def test_delta_rule_rows_behind_the_last_sequence(tail):
    lengths = [70, 30]
    x = make(lengths, 1, 2, 64, 64, torch.bfloat16, True, seed=tail, tail=tail)
    check_delta(x, lengths)
    check_delta(x, lengths, offsets="host")
    d = gpu(x)
    out = torch.full_like(d["v"], 7.0)
    off = torch.tensor([0, 70, 100], device="cuda", dtype=torch.int64)
    o, _ = ops.delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], offsets=off, initial_state=d["initial"], out=out)
    assert o.data_ptr() == out.data_ptr() and bool((out[100:] == 7).all()) and not bool((out[:100] == 7).all())


@pytest.mark.gpu
def test_delta_rule_no_tokens():
    x = gpu(make([0, 0], 1, 2, 64, 64, torch.float32, True))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    o, s = ops.delta_rule(*args, initial_state=x["initial"], offsets=[0, 0, 0])
    assert o.shape == (0, 2, 64) and torch.equal(s, x["initial"])
    got = ops.delta_rule_backward(x["do"], *args, initial_state=x["initial"], offsets=[0, 0, 0], d_final_state=x["ds"])
    assert torch.equal(got[5], x["ds"]) and got[0].shape == x["q"].shape
    _, s = ops.delta_rule(*args, offsets=[0, 0, 0])
    assert not s.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_delta_rule_decays_that_reset_and_that_hold(dtype):
    """g = -inf forgets the state before a token exactly; 0 keeps it; strong decays beside weak ones cost no digits."""
    lengths = [130]
    x = make(lengths, 1, 3, 64, 64, TYPES[dtype], True, seed=5)
    x["g"][:, 0] = 0.0
    x["g"][::17, 1] = -80.0
    x["g"][40, 2] = x["g"][64, 2] = x["g"][65, 2] = -math.inf
    check_delta(x, lengths, backward=False)
    # the backward pass against a reference that resets by a product with zero (e^-inf has no derivative to compare there)
    d = gpu(x)
    got = ops.delta_rule_backward(d["do"], d["q"], d["k"], d["v"], d["g"], d["beta"], initial_state=d["initial"])
    far = x["g"].clone()
    far[far == -math.inf] = -200.0
    near = ops.delta_rule_backward(d["do"], d["q"], d["k"], d["v"], far.cuda(), d["beta"], initial_state=d["initial"])
    for a, b in zip(got, near):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@pytest.mark.gpu
def test_delta_rule_beta_zero_and_two():
    lengths = [100]
    x = make(lengths, 1, 2, 64, 64, torch.float32, True, seed=9)
    x["beta"][:, 0] = 0.0
    x["beta"][::3, 1] = 0.0
    check_delta(x, lengths)
    x["beta"][:, 1] = 2.0          # reflections: lengths stay as they are
    x["g"][:] = 0.0
    check_delta(x, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_delta_rule_strided_broadcast_and_misaligned_inputs(dtype):
    t = TYPES[dtype]
    x = gpu(make([90], 2, 4, 64, 64, t, False, seed=11))
    want = ops.delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"])
    grads = ops.delta_rule_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["beta"])

    def same(q, k, v, g, beta, do):
        got = ops.delta_rule(q, k, v, g, beta)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(ops.delta_rule_backward(do, q, k, v, g, beta), grads))
    rows = torch.cat([x[n].reshape(90, -1) for n in ("q", "k", "v", "do")], 1)          # slices of one projection
    same(rows[:, :128].unflatten(1, (2, 64)), rows[:, 128:256].unflatten(1, (2, 64)), rows[:, 256:512].unflatten(1, (4, 64)),
         x["g"], x["beta"], rows[:, 512:].unflatten(1, (4, 64)))
    head_first = {n: x[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("q", "k", "v", "g", "beta", "do")}
    same(*(head_first[n] for n in ("q", "k", "v", "g", "beta", "do")))
    odd = {n: torch.cat([x[n].reshape(-1)[:1], x[n].reshape(-1)])[1:].view(x[n].shape) for n in ("q", "k", "v", "g", "beta", "do")}
    same(*(odd[n] for n in ("q", "k", "v", "g", "beta", "do")))
    last = {n: x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v", "do")}
    same(last["q"], last["k"], last["v"], x["g"], x["beta"], last["do"])
    one = x["k"][:1].expand(90, -1, -1)                                                   # the same key at every token
    a = ops.delta_rule(x["q"], one, x["v"], x["g"], x["beta"])
    b = ops.delta_rule(x["q"], one.contiguous(), x["v"], x["g"], x["beta"])
    assert all(torch.equal(p, r) for p, r in zip(a, b))


@pytest.mark.gpu
def test_delta_rule_nan_stays_in_its_sequence_and_head():
    lengths = [70, 80]
    x = make(lengths, 2, 2, 64, 64, torch.bfloat16, False, seed=13)
    d = gpu(x)
    off = torch.tensor(ends(lengths), dtype=torch.int32).cuda()
    o, s = ops.delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], offsets=off)
    v = d["v"].clone()
    v[66, 1, 3] = math.nan
    o2, s2 = ops.delta_rule(d["q"], d["k"], v, d["g"], d["beta"], offsets=off)
    assert torch.equal(o[:, 0], o2[:, 0]) and torch.equal(o[70:], o2[70:]) and torch.equal(s[1], s2[1])
    assert torch.equal(o[:64], o2[:64]) and bool(o2[66:70, 1, 3].isnan().all()) and bool(s2[0, 1, :, 3].isnan().all())


@pytest.mark.gpu
def test_delta_rule_gradients_against_differences():
    """Directional derivative of sum(o w) + sum(S ws) by central differences with two steps (the h^2 error removed)."""
    lengths = [70, 9]
    x = make(lengths, 1, 2, 64, 64, torch.float32, True, seed=17)
    d = gpu(x)
    off = torch.tensor(ends(lengths), dtype=torch.int32).cuda()
    names = ("q", "k", "v", "g", "beta")

    def loss(p, first):
        o, s = ops.delta_rule(*(p[n] for n in names), initial_state=first, offsets=off)
        return float((o.double() * d["do"].double()).sum() + (s.double() * d["ds"].double()).sum())
    got = ops.delta_rule_backward(d["do"], *(d[n] for n in names), initial_state=d["initial"], offsets=off, d_final_state=d["ds"])
    gen = torch.Generator().manual_seed(1)
    for i, name in enumerate(names + ("initial",)):
        # a direction along the gradient: its derivative is the gradient's length, well above the losses' own rounding
        way = got[i].cpu() / got[i].cpu().norm() + 0.1 * torch.nn.functional.normalize(
            torch.randn(got[i].shape, generator=gen).flatten(), dim=0).view(got[i].shape)
        way = way.cuda()
        slope = []
        for h in (2.0 ** -4, 2.0 ** -5):
            at = []
            for sign in (1, -1):
                p, first = dict(d), d["initial"]
                if name == "initial":
                    first = first + sign * h * way
                else:
                    p[name] = p[name] + sign * h * way
                at.append(loss(p, first))
            slope.append((at[0] - at[1]) / (2 * h))
        want = (4 * slope[1] - slope[0]) / 3
        have = float((got[i].double() * way.double()).sum())
        # fp32 losses of ~10^4 terms of size one over 2h: 100 x 2^-24 x 2^5 x a few; the h^4 term of Richardson's step: 2^-16
        assert abs(have - want) <= 2e-3 * abs(want) + 1e-3, (name, have, want)


@pytest.mark.gpu
def test_delta_rule_autograd():
    lengths = [40, 50]
    x = make(lengths, 1, 2, 64, 64, torch.bfloat16, True, seed=19)
    d = gpu(x)
    leaves = [d[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "beta")]
    first = d["initial"].clone().requires_grad_()
    o, s = ops.DeltaRule.apply(*leaves, None, first, ends(lengths))
    want = ops.delta_rule_backward(d["do"], *(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["initial"],
                                   offsets=ends(lengths), d_final_state=d["ds"])
    torch.autograd.backward([o, s], [d["do"], d["ds"]])
    for leaf, b in zip(leaves + [first], want):
        assert torch.equal(leaf.grad, b)
    o, _ = ops.DeltaRule.apply(*leaves, None, None, None)
    o.float().sum().backward()
    with torch.no_grad():
        assert ops.DeltaRule.apply(*leaves)[0].shape == d["v"].shape


# ----------------------------------------------------------------------------------------------------------------- step
def step_reference(x, state, slots, scale):
    state = state.double().clone()
    q, k, v, g, beta = (x[n].double() for n in ("q", "k", "v", "g", "beta"))
    group = v.shape[1] // q.shape[1]
    o = torch.zeros_like(v)
    for row, slot in enumerate(slots):
        if 0 <= slot < state.shape[0]:
            kr, qr = k[row].repeat_interleave(group, 0), q[row].repeat_interleave(group, 0)
            S = state[slot] * g[row].exp()[:, None, None]
            u = beta[row][:, None] * (v[row] - (kr[:, None] @ S)[:, 0])
            state[slot] = S + kr[:, :, None] * u[:, None]
            o[row] = scale * (qr[:, None] @ state[slot])[:, 0]
        elif slot != -1:
            o[row] = math.nan
    return o, state


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, hk, hv, dk, dv, rows, pool", [
    ("bf16", 1, 1, 128, 128, 1, 1), ("fp32", 2, 4, 64, 64, 5, 9), ("fp16", 1, 3, 128, 192, 7, 7), ("bf16", 2, 2, 64, 256, 33, 70),
])
def test_delta_step(dtype, hk, hv, dk, dv, rows, pool):
    x = make([rows], hk, hv, dk, dv, TYPES[dtype], False, seed=rows)
    gen = torch.Generator().manual_seed(rows)
    state = torch.randn(pool, hv, dk, dv, generator=gen) * 0.3
    for slots in (None, torch.randperm(pool, generator=gen)[:rows].to(torch.int32)):
        want_o, want = step_reference(x, state, range(rows) if slots is None else slots.tolist(), x["scale"])
        d, s = gpu(x), state.cuda()
        o = ops.delta_rule_step(d["q"], d["k"], d["v"], d["g"], d["beta"], s, slots=None if slots is None else slots.cuda())
        close("o", o, want_o, dk)
        close("state", s, want, dk)


@pytest.mark.gpu
def test_delta_step_padded_rows_repeated_slots_and_bad_ones():
    rows = 300
    x = make([rows], 1, 2, 64, 64, torch.float32, False, seed=2)
    state = torch.randn(40, 2, 64, 64, generator=torch.Generator().manual_seed(2))
    slots = [(i * 7) % 40 for i in range(60)] + [-1] * 100 + [5] * 20 + [40, -2, 2 ** 31 - 1, -2 ** 31] + [39] + [-1] * 115
    want_o, want = step_reference(x, state, slots, x["scale"])
    d, s = gpu(x), state.cuda()
    o = ops.delta_rule_step(d["q"], d["k"], d["v"], d["g"], d["beta"], s, slots=torch.tensor(slots, dtype=torch.int32).cuda())
    bad = want_o.isnan()
    assert torch.equal(o.isnan().cpu(), bad) and bad.any()
    close("o", o.cpu().masked_fill(bad, 0.0), want_o.masked_fill(bad, 0.0), 64, chunks=6)
    close("state", s, want, 64, chunks=6)
    out = torch.full((rows, 2, 2, 64), 3.0, device="cuda")[:, 1]
    s2 = state.cuda()
    got = ops.delta_rule_step(d["q"], d["k"], d["v"], d["g"], d["beta"], s2, slots=torch.tensor(slots, dtype=torch.int32).cuda(), out=out)
    assert torch.equal(got.nan_to_num(9.0), o.nan_to_num(9.0)) and torch.equal(s2, s)
    assert bool((out._base[:, 0] == 3).all())


@pytest.mark.gpu
def test_delta_step_strided_pool_and_no_rows():
    x = gpu(make([3], 1, 2, 64, 64, torch.bfloat16, False, seed=4))
    big = torch.randn(6, 2, 2, 64, 64, device="cuda")
    state = big[:, 1]
    plain = state.clone()
    rest = big[:, 0].clone()
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    a = ops.delta_rule_step(*args, state)
    b = ops.delta_rule_step(*args, plain)
    assert torch.equal(a, b) and torch.equal(state, plain) and torch.equal(big[:, 0], rest)
    none = tuple(t[:0] for t in args)
    assert ops.delta_rule_step(*none, plain).shape == (0, 2, 64)
    assert ops.delta_rule_step(*none, plain[:0]).shape == (0, 2, 64)


@pytest.mark.gpu
def test_delta_step_goes_on_where_a_sequence_ended():
    """What serving does: a prompt through delta_rule, its state into the pool, then tokens one by one -- the same as the whole."""
    x = gpu(make([80], 1, 2, 128, 128, torch.float32, False, seed=6))
    names = ("q", "k", "v", "g", "beta")
    o, s = ops.delta_rule(*(x[n] for n in names))
    first, state = ops.delta_rule(*(x[n][:70] for n in names))
    pool = torch.zeros(4, 2, 128, 128, device="cuda")
    pool[2] = state[0]
    slot = torch.tensor([2], dtype=torch.int32, device="cuda")
    rest = [ops.delta_rule_step(*(x[n][t:t + 1] for n in names), pool, slots=slot) for t in range(70, 80)]
    got = torch.cat([first] + rest)
    close("o", got, o.double().cpu(), 256, chunks=2)
    close("state", pool[2:3], s.double().cpu(), 256, chunks=2)
    assert not pool[:2].any() and not pool[3].any()


# ----------------------------------------------------------------------------------------------------------- layer norm
def norm_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / (((x - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    return h * (1 if w is None else w.double()) + (0 if b is None else b.double()), mean[..., 0], rstd[..., 0], h


def check_norm(x, w, b, dy, eps=1e-5, strided=None):
    y, mean, rstd = ops.layer_norm(x, w, b, eps)
    ry, rmean, rrstd, h = norm_reference(x.cpu(), None if w is None else w.cpu(), None if b is None else b.cpu(), eps)
    n = x.shape[-1]
    close("y", y, ry, n)
    # the mean is off by u of the sum's magnitude, not of its own size
    assert float((mean.cpu().double() - rmean).abs().max()) <= 8 * n * U * float(x.abs().double().max())
    close("rstd", rstd, rrstd, n)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    g = dy.cpu().double()
    e = g * (1 if w is None else w.cpu().double())
    want = rrstd[..., None] * (e - e.mean(-1, keepdim=True) - h * (e * h).mean(-1, keepdim=True))
    scale = float((rrstd[..., None] * e).abs().max())      # where dx cancels, it is off by u of what cancelled
    off = (dx.cpu().double() - want).abs()
    assert bool((off <= (half(dx.dtype) if dx.dtype != torch.float32 else U) * want.abs() + 8 * n * U * scale).all()), float(off.max())
    rows = g.reshape(-1, n).shape[0]
    lead = tuple(range(g.dim() - 1))
    for name, a, r, mag in (("dw", dw, (g * h).sum(lead) if lead else g * h, (g * h).abs()), ("db", db, g.sum(lead) if lead else g, g.abs())):
        if a is None:
            continue
        mag = mag.sum(lead) if lead else mag
        tol = (half(a.dtype) if a.dtype != torch.float32 else U) * r.abs() + 8 * (rows + n) * U * mag
        assert a.shape == r.shape and bool(((a.cpu().double() - r).abs() <= tol).all()), name
    again = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(again[0], dx) and torch.equal(again[2], db) and (dw is None or torch.equal(again[1], dw))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, wtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("rows, width", [(1, 1), (5, 7), (100, 128), (33, 129), (17, 300), (9, 512), (70, 1000), (3, 1025),
                                         (5, 2049), (4, 4099), (3, 8192), (5, 9001)])
def test_layer_norm(dtype, wtype, rows, width):
    gen = torch.Generator().manual_seed(rows * width)
    x = (torch.randn(rows, width, generator=gen) * 2 + 3).to(TYPES[dtype]).cuda()
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(TYPES[wtype]).cuda()
    b = (0.2 * torch.randn(width, generator=gen)).to(TYPES[wtype]).cuda()
    dy = torch.randn(rows, width, generator=gen).to(TYPES[dtype]).cuda()
    check_norm(x, w, b, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layer_norm_strides_shapes_and_no_weight(dtype):
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(1)
    big = torch.randn(6, 50, 3, 200, generator=gen).to(t).cuda()
    dy = torch.randn(6, 50, 200, generator=gen).to(t).cuda()
    w = torch.randn(200, generator=gen).to(t).cuda()
    check_norm(big[:, :, 1], w, None, dy)                                  # no single row stride: copied
    check_norm(big[0, :, 1], None, None, dy[0])                            # strided rows
    check_norm(big[0, :, 1, 3:], None, w[3:], dy[0, :, 3:])                # misaligned rows
    check_norm(big[0, :, :, 5].transpose(0, 1), w[:50], None, dy[0, :3, :50])  # strided last dimension
    check_norm(big[0, 0, 0], w, w, dy[0, 0])                               # one row without a batch dimension
    out = torch.full((50, 2, 200), 5.0, device="cuda", dtype=t)
    y, _, _ = ops.layer_norm(big[0, :, 1], w, out=out[:, 1])
    assert torch.equal(y, ops.layer_norm(big[0, :, 1], w)[0]) and bool((out[:, 0] == 5).all())


@pytest.mark.gpu
def test_layer_norm_constant_rows_and_no_rows():
    x = torch.full((4, 300), 1000.0, device="cuda")
    y, mean, rstd = ops.layer_norm(x, eps=1e-5)
    assert not y.any() and bool((mean == 1000).all()) and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))
    x = torch.zeros(0, 33, device="cuda")
    w = torch.ones(33, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w)
    dx, dw, db = ops.layer_norm_backward(x, x, w, mean, rstd)
    assert y.shape == x.shape and dx.shape == x.shape and not dw.any() and not db.any()
    x = torch.randn(5, 64, device="cuda")
    x[2, 7] = math.inf
    x[3, 9] = math.nan
    y, mean, rstd = ops.layer_norm(x)
    assert bool(y[[0, 1, 4]].isfinite().all()) and bool(y[[2, 3]].isnan().any(1).all())


@pytest.mark.gpu
def test_layer_norm_autograd_and_differences():
    gen = torch.Generator().manual_seed(8)
    x, dy = (torch.randn(7, 96, generator=gen).cuda() for _ in range(2))
    w, b = (torch.randn(96, generator=gen).cuda() for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.LayerNorm.apply(*leaves).backward(dy)
    _, mean, rstd = ops.layer_norm(x, w, b)
    for leaf, want in zip(leaves, ops.layer_norm_backward(dy, x, w, mean, rstd)):
        assert torch.equal(leaf.grad, want)
    for i in range(3):
        way = torch.nn.functional.normalize(leaves[i].grad.flatten(), dim=0).view(leaves[i].shape)
        slope = []
        for h in (2.0 ** -4, 2.0 ** -5):
            at = []
            for sign in (1, -1):
                p = [x, w, b]
                p[i] = p[i] + sign * h * way
                at.append(float((ops.layer_norm(*p)[0].double() * dy.double()).sum()))
            slope.append((at[0] - at[1]) / (2 * h))
        want = (4 * slope[1] - slope[0]) / 3
        have = float((leaves[i].grad.double() * way.double()).sum())
        assert abs(have - want) <= 1e-3 * abs(want) + 1e-3, (i, have, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, rows, width", [("bf16", 20000, 16), ("fp32", 5000, 300), ("fp16", 4200, 130), ("bf16", 4100, 1030),
                                                ("bf16", 700, 9001), ("fp32", 600, 4100)])
def test_layer_norm_more_rows_than_workgroups(dtype, rows, width):
    gen = torch.Generator().manual_seed(rows + width)
    x, dy = (torch.randn(rows, width, generator=gen).to(TYPES[dtype]).cuda() for _ in range(2))
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(TYPES[dtype]).cuda()
    check_norm(x, w, w, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [33, 20000])
def test_layer_norm_in_place_and_wide_without_rows(width):
    x = torch.randn(7, width, generator=torch.Generator().manual_seed(width)).cuda()
    want = ops.layer_norm(x)
    got = ops.layer_norm(x, out=x)
    assert got[0].data_ptr() == x.data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want))
    none, w = x[:0], torch.ones(width, device="cuda")
    y, mean, rstd = ops.layer_norm(none, w)
    dx, dw, db = ops.layer_norm_backward(none, none, w, mean, rstd)
    assert y.shape == dx.shape == (0, width) and not dw.any() and not db.any()


# ------------------------------------------------------------------------------------------------------------- together
def layer(x, p, offsets=None, state=None):
    """A recurrent layer as a user builds it: norm, projections, the delta rule, the heads' norm, projection back, residual."""
    n = x.shape[0]
    y, _, _ = ops.layer_norm(x, p["w1"], p["b1"])
    z = y @ p["in"]
    q = torch.nn.functional.normalize(z[:, :128].unflatten(1, (2, 64)).float(), dim=-1).to(x.dtype)
    k = torch.nn.functional.normalize(z[:, 128:256].unflatten(1, (2, 64)).float(), dim=-1).to(x.dtype)
    v = z[:, 256:512].unflatten(1, (4, 64))
    g = -torch.nn.functional.softplus((y @ p["g"]).float())
    beta = torch.sigmoid((y @ p["beta"]).float())
    if state is not None:
        o = ops.delta_rule_step(q, k, v, g, beta, state)
    else:
        o, last = ops.delta_rule(q, k, v, g, beta, offsets=offsets)
    o, _, _ = ops.layer_norm(o, p["w2"])
    out = x + o.reshape(n, 256) @ p["out"]
    return out if state is not None else (out, last)


def parameters(dtype):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: (torch.randn(*s, generator=gen) / math.sqrt(s[0])).to(dtype).cuda()  # noqa: E731
    return {"w1": (1 + r(200)), "b1": r(200), "in": r(200, 512), "g": r(200, 4), "beta": r(200, 4), "w2": 1 + r(64), "out": r(256, 200)}


@pytest.mark.gpu
def test_layers_over_a_prompt_and_then_token_by_token():
    p = parameters(torch.float32)
    x = torch.randn(90, 200, generator=torch.Generator().manual_seed(1)).cuda()
    whole, _ = layer(x, p)
    first, state = layer(x[:70], p)
    rest = [layer(x[t:t + 1], p, state=state) for t in range(70, 90)]
    got = torch.cat([first] + rest)
    # the projections before and behind are sums of 200 and 256 products in another order: n u of magnitudes below ten
    assert float((got - whole).abs().max()) <= 10 * 8 * (200 + 256 + 192) * U


@pytest.mark.gpu
def test_calls_on_two_streams_and_into_graphs():
    """Two streams at once, and two captured graphs replayed several times with eager work between: the eager results."""
    sets = [make([70, 130], 2, 4, 64, 64, torch.bfloat16, True, seed=s) for s in (1, 2)]
    off = torch.tensor([0, 70, 200], dtype=torch.int32).cuda()
    w = torch.randn(64, generator=torch.Generator().manual_seed(3)).cuda()

    def work(d):
        o, s, saved = ops.delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_state=d["initial"], offsets=off, keep=True)
        grads = ops.delta_rule_backward(d["do"], d["q"], d["k"], d["v"], d["g"], d["beta"], initial_state=d["initial"],
                                        offsets=off, d_final_state=d["ds"], saved=saved)
        y, mean, rstd = ops.layer_norm(o, w)
        dn = ops.layer_norm_backward(d["do"], o, w, mean, rstd)
        pool = d["pool"].clone()
        t = ops.delta_rule_step(d["q"][:8], d["k"][:8], d["v"][:8], d["g"][:8], d["beta"][:8], pool)
        return (o, s) + grads + (y, mean, rstd) + dn + (t, pool)

    ds = [dict(gpu(x), pool=torch.randn(8, 4, 64, 64, generator=torch.Generator().manual_seed(i)).cuda()) for i, x in enumerate(sets)]
    want = [[t.clone() for t in work(d)] for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, d in zip(streams, ds):
            with torch.cuda.stream(st):
                got.append(work(d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for d in ds:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(d))
        graphs.append(graph)
    for turn in range(3):
        for graph in graphs if turn != 1 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), turn
        assert all(torch.equal(x, y) for x, y in zip(work(ds[turn % 2]), want[turn % 2]))
    # other inputs in the captured buffers
    ds[0]["v"].copy_(ds[1]["v"])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], work(ds[0])))


@pytest.mark.gpu
def test_autograd_forms_refuse_capture():
    x = gpu(make([10], 1, 1, 64, 64, torch.float32, False))
    leaf = x["v"].clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x["v"] * 2
        with pytest.raises(RuntimeError, match="captured"):
            ops.DeltaRule.apply(x["q"], x["k"], leaf, x["g"], x["beta"])
        with pytest.raises(RuntimeError, match="captured"):
            ops.LayerNorm.apply(leaf)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x["v"] * 2)


# ------------------------------------------------------------------------------------------------- one arithmetic for all types
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hk, hv, dk, dv, lengths", [
    (1, 2, 128, 128, [1, 200, 65]), (2, 4, 64, 64, [130, 33]), (1, 1, 128, 256, [300]),          # few chains
    (4, 8, 128, 128, [70, 64, 1, 131, 33]), (16, 16, 64, 64, [70, 64, 1, 131, 33]),               # more than compute units
])
def test_delta_rule_of_16_bits_is_the_fp32_one_rounded_once(dtype, hk, hv, dk, dv, lengths):
    """Every product takes the same terms whatever the type of q, k, v and d_o (those that a 16-bit value lacks are zeros), so
    the same values in float32 give the same sums: o, dq, dk and dv are those of float32 rounded once, the rest is equal.  (What
    `close` leaves a 16-bit o beside its rounding, two terms an operand, is therefore not used.)"""
    x = gpu(make(lengths, hk, hv, dk, dv, TYPES[dtype], True, seed=dk + dv))
    off = torch.tensor(ends(lengths), dtype=torch.int32).cuda()

    def run(widen):
        q, k, v, do = (x[n].float() if widen else x[n] for n in ("q", "k", "v", "do"))
        args, kw = (q, k, v, x["g"], x["beta"]), dict(initial_state=x["initial"], offsets=off)
        o, s, saved = ops.delta_rule(*args, keep=True, **kw)
        return (o, s) + ops.delta_rule(*args, **kw) + ops.delta_rule_backward(do, *args, d_final_state=x["ds"], saved=saved, **kw)
    names = ("o", "final_state", "o", "final_state", "dq", "dk", "dv", "dg", "dbeta", "d_initial")
    for name, a, b in zip(names, run(False), run(True)):
        assert torch.equal(a, b.to(a.dtype)), (name, float((a.double() - b.double()).norm() / b.double().norm()))


# ------------------------------------------------------------------------------------------- written in place, and autograd
def test_what_is_written_in_place_may_not_require_a_gradient():
    x = make([4], 1, 1, 64, 64, torch.float32, False)
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    leaf = torch.zeros(4, 1, 64, requires_grad=True)
    state = torch.zeros(4, 1, 64, 64)
    calls = [lambda: ops.delta_rule(*args, out=leaf), lambda: ops.delta_rule(*args, out=leaf * 2),
             lambda: ops.delta_rule_step(*args, state, out=leaf), lambda: ops.layer_norm(x["v"], out=leaf),
             lambda: ops.delta_rule_step(*args, state.clone().requires_grad_()), lambda: ops.layer_norm(leaf * 1, out=leaf[:])]
    for call in calls:
        with pytest.raises(RuntimeError, match="written in place"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.gpu
def test_autograd_sees_what_is_written_in_place():
    x = gpu(make([10], 1, 2, 64, 64, torch.float32, False, seed=23))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])

    def spoiled(t, write):
        """A backward pass that needs t as it was has to fail after `write`, and says why."""
        w = torch.ones(t.shape[-1], device="cuda", requires_grad=True)
        z = (w * t).sum()
        before = t._version
        write()
        assert t._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    out = torch.randn(10, 2, 64, device="cuda")
    spoiled(out, lambda: ops.delta_rule(*args, out=out))
    spoiled(out, lambda: ops.delta_rule_step(*args, torch.zeros(10, 2, 64, 64, device="cuda"), out=out))
    spoiled(out, lambda: ops.layer_norm(x["v"], out=out))
    spoiled(out, lambda: ops.layer_norm(out, out=out))
    spoiled(out, lambda: ops.layer_norm(out[:, 0], out=out[:, 0]))
    state = torch.zeros(10, 2, 64, 64, device="cuda")
    spoiled(state, lambda: ops.delta_rule_step(*args, state))
    rows, w = x["v"][:, 0].clone(), torch.ones(64, device="cuda", requires_grad=True)
    y = ops.LayerNorm.apply(rows, w)
    ops.layer_norm(rows, out=rows)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # gradients that do not need what was overwritten are as they were
    leaf = torch.randn(10, 2, 64, 64, device="cuda", requires_grad=True)
    pool = leaf * 2
    with torch.no_grad():
        ops.delta_rule_step(*args, pool)
    pool.sum().backward()
    assert bool((leaf.grad == 2).all())


def test_plain_calls_refuse_inputs_that_require_a_gradient():
    """They cannot be followed by autograd: without a refusal the gradient of such an input would silently be missing."""
    x = make([4], 1, 1, 64, 64, torch.float32, True)
    names = ("q", "k", "v", "g", "beta")
    plain = [x[n] for n in names]
    calls = []
    for i in range(5):
        args = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(plain)]
        calls += [("DeltaRule.apply", lambda a=args: ops.delta_rule(*a)), ("delta_rule_step", lambda a=args: ops.delta_rule_step(*a, torch.zeros(4, 1, 64, 64)))]
    calls += [("DeltaRule.apply", lambda: ops.delta_rule(*plain, initial_state=x["initial"].clone().requires_grad_())),
              ("DeltaRule.apply", lambda: ops.delta_rule(plain[0].clone().requires_grad_() * 2, *plain[1:], keep=True))]
    w = torch.ones(64, requires_grad=True)
    calls += [("LayerNorm.apply", lambda: ops.layer_norm(x["v"].clone().requires_grad_())), ("LayerNorm.apply", lambda: ops.layer_norm(x["v"], w)),
              ("LayerNorm.apply", lambda: ops.layer_norm(x["v"], None, w))]
    for match, call in calls:
        with pytest.raises(RuntimeError, match=match):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
        with torch.inference_mode(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.gpu
def test_autograd_forms_are_captured_where_nothing_is_recorded():
    """Under no_grad, and without an input that requires a gradient: nothing to record, so the plain calls."""
    x = gpu(make([70, 10], 1, 2, 64, 64, torch.bfloat16, True, seed=29))
    off = torch.tensor([0, 70, 80], dtype=torch.int32, device="cuda")
    w = torch.randn(64, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "beta")]
    plain = [x[n] for n in ("q", "k", "v", "g", "beta")]
    with torch.no_grad():
        want = ops.delta_rule(*plain, initial_state=x["initial"], offsets=off)
        want += ops.layer_norm(want[0], w)[:1]

    def under_no_grad():
        with torch.no_grad():
            o, s = ops.DeltaRule.apply(*leaves, None, x["initial"], off)
            return o, s, ops.LayerNorm.apply(o, w)

    def without_leaves():
        o, s = ops.DeltaRule.apply(*plain, None, x["initial"], off)
        return o, s, ops.LayerNorm.apply(o, w.detach())
    for call in (under_no_grad, without_leaves):
        got = call()
        assert not any(t.requires_grad for t in got) and all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for _ in range(3):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert all(torch.equal(a, b) for a, b in zip(call(), want))
    # with gradients recorded all five and the state's are there, and for one leaf alone its own
    o, s = ops.DeltaRule.apply(*leaves, None, x["initial"], off)
    o.backward(x["do"])
    grads = ops.delta_rule_backward(x["do"], *plain, initial_state=x["initial"], offsets=off)
    assert all(torch.equal(t.grad, b) for t, b in zip(leaves, grads))
    beta = x["beta"].clone().requires_grad_()
    ops.DeltaRule.apply(*plain[:4], beta, None, x["initial"], off)[0].backward(x["do"])
    assert torch.equal(beta.grad, grads[4])


# ---------------------------------------------------------------------------------------------------- how much one call takes
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype, width, rows, text", [
    (1, 64, 2 ** 24, b"null"), (0, 4096, 2 ** 24, b"null"), (1, 8192, 2 ** 24, b"null"), (1, 128, 2 ** 36 - 1, b"null"),
    (1, 128, 2 ** 36, b"more than one call"), (0, 4097, 2 ** 24 - 1, b"null"), (0, 4097, 2 ** 24, b"more than one call"),
    (2, 8193, 2 ** 24, b"more than one call"),
])
def test_layer_norm_takes_rows_up_to_its_kernels_limits(backward, dtype, width, rows, text):
    lib = _lib.load()
    c = _lib.HelenLayerNormC()
    c.struct_size = ctypes.sizeof(c)
    c.dtype, c.weight_dtype, c.width, c.rows, c.eps = dtype, dtype, width, rows, 1e-5
    rc = lib.helen_layer_norm_backward(ctypes.byref(c), None, 0, None) if backward else lib.helen_layer_norm_forward(ctypes.byref(c), None)
    assert rc == -1 and text in lib.helen_last_error(), lib.helen_last_error()


@pytest.mark.gpu
def test_layer_norm_of_more_than_2_24_rows():
    """Rows do not depend on each other: those of one call are those of two, and the sums over all rows those of 64 bits."""
    rows, width, cut = 2 ** 24 + 5, 16, 2 ** 23 + 1
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(rows, width, generator=gen, device="cuda").bfloat16() for _ in range(2))
    w, b = (torch.randn(width, generator=gen, device="cuda") for _ in range(2))
    y, mean, rstd = ops.layer_norm(x, w, b)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    for part in (slice(0, cut), slice(cut, rows)):
        got = ops.layer_norm(x[part], w, b)
        assert all(torch.equal(p, q[part]) for p, q in zip(got, (y, mean, rstd)))
        assert torch.equal(ops.layer_norm_backward(dy[part], x[part], w, *got[1:])[0], dx[part])
    sums = torch.zeros(4, width, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 2 ** 21):
        g, h = dy[at:at + 2 ** 21].double(), (x[at:at + 2 ** 21].double() - mean[at:at + 2 ** 21, None]) * rstd[at:at + 2 ** 21, None]
        sums += torch.stack([(g * h).sum(0), (g * h).abs().sum(0), g.sum(0), g.abs().sum(0)])
    # a column's sum passes a lane (rows over 512 x 16 of them), 16 lanes, 512 workgroups one after another; h itself is off by 3 u
    n = rows / (512 * 16) + 16 + 512 + 3
    for got, want, size in ((dw, sums[0], sums[1]), (db, sums[2], sums[3])):
        assert bool(((got.double() - want).abs() <= n * U * size + U * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, width", [("bf16", 2 ** 24 + 3), ("bf16", 2 ** 26 + 37)])
def test_layer_norm_gradient_of_very_wide_rows(dtype, width):
    """The sums over the rows of more columns than one launch has threads for (64 threads a column and gradient); one row, so
    they are dy h and dy themselves."""
    gen = torch.Generator(device="cuda").manual_seed(width)
    x, dy = (torch.randn(1, width, generator=gen, device="cuda").to(TYPES[dtype]) for _ in range(2))
    w = torch.ones(width, device="cuda", dtype=TYPES[dtype])
    mean, rstd = torch.tensor([0.25], device="cuda"), torch.tensor([0.5], device="cuda")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(db, dy[0])
    # x - 1/4 and its half are rounded to 24 bits at most once, the product too, and dw to its own type
    want = dy[0].double() * (x[0].double() - 0.25) * 0.5
    assert bool(((dw.double() - want).abs() <= (half(dw.dtype) + 3 * U) * want.abs() + 1e-38).all())
    assert bool(dx.isfinite().all())


@pytest.mark.parametrize("change, backward, text", [
    # 64 tokens a slot: 9,000,002 slots fit launches of 256 threads a slot and key head, but not the gradients' 512 (width_k 128)
    (dict(tokens=576000000, heads_k=1, heads_v=1), False, b"null input"),
    (dict(tokens=576000000, heads_k=1, heads_v=1), True, b"more than one call"),
    (dict(tokens=576000000, heads_k=1, heads_v=1, width_k=64), True, b"null input"),
    (dict(tokens=1152000000, heads_k=1, heads_v=1), False, b"more than one call"),
    # 4 x 2^22 groups of 32 columns, less the room for rounding up, and one sequence more
    (dict(tokens=0, sequences=2 ** 22 - 2, heads_k=1, heads_v=1, offsets=4096), False, b"workspace"),
    (dict(tokens=0, sequences=2 ** 22, heads_k=1, heads_v=1, offsets=4096), False, b"more than one call"),
    (dict(tokens=0, sequences=2 ** 31 - 2, heads_k=2 ** 30, heads_v=2 ** 30, offsets=4096), False, b"more than one call"),
])
def test_delta_rule_takes_what_its_launches_can_count(change, backward, text):
    lib = _lib.load()
    c = ctypes.byref(description(**change))
    rc = lib.helen_delta_rule_backward(c, None, 0, None, 0, None) if backward else lib.helen_delta_rule_forward(c, 0, None, 0, None)
    assert rc == -1 and text in lib.helen_last_error(), lib.helen_last_error()


def test_delta_step_refuses_more_rows_than_its_launch_can_count():
    lib = _lib.load()
    c = _lib.HelenDeltaStepC()
    c.struct_size = ctypes.sizeof(c)
    c.heads_k, c.heads_v, c.width_k, c.width_v, c.rows, c.pool = 1, 2 ** 30, 128, 256, 2 ** 30, 2 ** 30
    assert lib.helen_delta_rule_step(ctypes.byref(c), None) == -1
    assert b"more than one call" in lib.helen_last_error(), lib.helen_last_error()


# ----------------------------------------------------------------------------------------- resets, long chains, equal lengths
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("lengths, heads, decay", [([130], 3, 1.0), ([200, 1, 64], 3, 25.0), ([70, 64, 1, 131, 33], 16, 1.0)])
def test_delta_rule_gradients_at_resets_and_strong_decays(dtype, lengths, heads, decay):
    """All gradients against the reference where the state is held (g = 0), all but forgotten (-80) and forgotten: e^-200 has a
    derivative in 64 bits, and is as good as zero there.  -inf in its place gives the same bits.  (16 heads of 5 sequences: 320
    chains, the kernel for many.)"""
    x = make(lengths, 1 if heads == 3 else 16, heads, 64, 64, TYPES[dtype], True, seed=31, decay=decay)
    x["g"][:, 0] = 0.0
    x["g"][::17, 1] = -80.0
    far = torch.zeros(x["g"].shape, dtype=torch.bool)
    far[0, 2] = far[40, 2] = far[64, 2] = far[65, 2] = far[-1, 2] = True
    x["g"][far] = -200.0
    check_delta(x, lengths)
    d = gpu(x)
    off = torch.tensor(ends(lengths), dtype=torch.int32, device="cuda")

    def run(g):
        args, kw = (d["q"], d["k"], d["v"], g, d["beta"]), dict(initial_state=d["initial"], offsets=off)
        o, s, saved = ops.delta_rule(*args, keep=True, **kw)
        return (o, s) + ops.delta_rule_backward(d["do"], *args, d_final_state=d["ds"], saved=saved, **kw)
    near = run(d["g"])
    for a, b in zip(run(d["g"].masked_fill(far.cuda(), -math.inf)), near):
        assert torch.equal(a, b)
    assert not near[5][0, 2].any()            # a reset before the first token: the initial state has no part in anything


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lengths", [[2600, 1111], [2600] + [3] * 50], ids=["few chains", "many chains"])
def test_delta_rule_long_chains(dtype, lengths):
    """41 chunks in a row, with the kernels for few chains (24 of 16 columns) and for many (612).  Head 0 never forgets (g = 0): an
    error made in a chunk may stay, so the bounds count all chunks.  The slowest other head decays by e^-0.025|N| a token, e^-1.3 a
    chunk on average: beside what a chunk adds, what is left of those before it makes up 1 / (e^1.3 - 1) = 0.4 of it, so two are
    counted.  The float32 results (state, dg, dbeta, d_initial) are held to that without a rounding to hide in."""
    hv, count = 3, 41
    x = make(lengths, 1, hv, 64, 64, TYPES[dtype], True, seed=len(lengths))
    n = x["g"].shape[0]
    x["g"] = -torch.randn(n, hv, generator=torch.Generator().manual_seed(5)).abs() * torch.tensor([0.0, 0.025, 0.5])
    d = gpu(x)
    off = torch.tensor(ends(lengths), dtype=torch.int32, device="cuda")
    args, kw = (d["q"], d["k"], d["v"], d["g"], d["beta"]), dict(scale=x["scale"], initial_state=d["initial"], offsets=off)
    o, s, saved = ops.delta_rule(*args, keep=True, **kw)
    got = (o, s) + ops.delta_rule_backward(d["do"], *args, d_final_state=d["ds"], saved=saved, **kw)
    assert all(torch.equal(a, b) for a, b in zip(ops.delta_rule(*args, **kw), got))
    leaves = [x[m].double().requires_grad_() for m in ("q", "k", "v", "g", "beta")]
    # dq and dk are summed over the heads: here they are wanted a head at a time, so every head gets keys of its own
    leaves[0], leaves[1] = (t.detach().repeat_interleave(hv, 1).requires_grad_() for t in leaves[:2])
    first = x["initial"].double().requires_grad_()
    ro, rs = delta_reference(*leaves, x["scale"], first, lengths)
    loss = (ro * x["do"].double()).sum() + (rs * x["ds"].double()).sum()
    want = dict(zip(("o", "final_state", "dq", "dk", "dv", "dg", "dbeta", "d_initial"),
                    (ro, rs) + torch.autograd.grad(loss, leaves + [first])))
    products = 64 + 64 + 64
    for name, a in zip(("o", "final_state", "dq", "dk", "dv", "dg", "dbeta", "d_initial"), got):
        b = want[name]
        if name in ("dq", "dk"):
            close(name, a, b.sum(1, keepdim=True), products, count)
            continue
        for head, chunks in ((slice(0, 1), count), (slice(1, hv), 2)):
            close("%s of heads %s" % (name, head), a[:, head], b[:, head], products, chunks)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences, length, hk, hv", [(3, 70, 1, 2), (40, 33, 2, 4), (2, 64, 1, 1), (7, 1, 1, 2)])
def test_delta_rule_sequences_of_one_length_without_offsets(sequences, length, hk, hv):
    """The C entries with offsets NULL: the results of the same call with offsets, bit for bit."""
    dk = dv = 64
    lengths = [length] * sequences
    x = gpu(make(lengths, hk, hv, dk, dv, torch.bfloat16, True, seed=sequences))
    tokens = sequences * length
    off = torch.tensor(ends(lengths), dtype=torch.int32, device="cuda")
    args, kw = (x["q"], x["k"], x["v"], x["g"], x["beta"]), dict(scale=x["scale"], initial_state=x["initial"], offsets=off)
    o, s, saved = ops.delta_rule(*args, keep=True, **kw)
    want = (o, s) + ops.delta_rule_backward(x["do"], *args, d_final_state=x["ds"], saved=saved, **kw)
    lib = _lib.load()
    c = _lib.HelenDeltaRuleC()
    c.struct_size, c.device, c.dtype = ctypes.sizeof(c), x["q"].get_device(), _lib.HELEN_TYPE_BF16
    c.heads_k, c.heads_v, c.width_k, c.width_v, c.tokens, c.sequences, c.scale = hk, hv, dk, dv, tokens, sequences, x["scale"]
    sizes = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(lib.helen_delta_rule_bytes(ctypes.byref(c), *(ctypes.byref(t) for t in sizes)))
    plain, kept, own = (torch.empty(t.value, dtype=torch.uint8, device="cuda") for t in sizes)
    got = [torch.full_like(t, 7.0) for t in want]
    pair = lambda t: (ctypes.c_int64 * 2)(*t.stride()[:2])  # noqa: E731
    for name, t in zip(("q", "k", "v", "g", "beta"), args):
        setattr(c, name, t.data_ptr())
        setattr(c, name + "_stride", pair(t))
    c.initial_state, c.d_o, c.d_o_stride, c.d_final_state = x["initial"].data_ptr(), x["do"].data_ptr(), pair(x["do"]), x["ds"].data_ptr()
    c.o, c.o_stride, c.final_state = got[0].data_ptr(), pair(got[0]), got[1].data_ptr()
    for name, t in zip(("grad_q", "grad_k", "grad_v", "grad_g", "grad_beta", "grad_initial_state"), got[2:]):
        setattr(c, name, t.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    call = ctypes.byref(c)
    _lib.check(lib.helen_delta_rule_forward(call, 0, plain.data_ptr(), plain.numel(), stream))
    assert torch.equal(got[0], o) and torch.equal(got[1], s)
    got[0].fill_(7.0)
    _lib.check(lib.helen_delta_rule_forward(call, 1, kept.data_ptr(), kept.numel(), stream))
    _lib.check(lib.helen_delta_rule_backward(call, kept.data_ptr(), kept.numel(), own.data_ptr(), own.numel(), stream))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_delta_rule_under_a_checkpoint_keeps_nothing_and_has_the_same_gradients():
    from torch.utils.checkpoint import checkpoint
    x = gpu(make([640], 2, 4, 128, 128, torch.bfloat16, True, seed=37))
    names = ("q", "k", "v", "g", "beta")
    grads, held = [], []
    for again in (False, True):
        leaves = [x[n].clone().requires_grad_() for n in names] + [x["initial"].clone().requires_grad_()]
        before = torch.cuda.memory_allocated()
        if again:
            o, s = checkpoint(lambda *a: ops.DeltaRule.apply(*a[:5], None, a[5]), *leaves, use_reentrant=False)
        else:
            o, s = ops.DeltaRule.apply(*leaves[:5], None, leaves[5])
        held.append(torch.cuda.memory_allocated() - before)
        torch.autograd.backward([o, s], [x["do"], x["ds"]])
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    kept = ops._rule_bytes(_lib.HELEN_TYPE_BF16, 2, 4, 128, 128, 640, 1)[1]
    assert held[0] - held[1] >= kept


# ------------------------------------------------------------------------------------------------ calls that the documents allow
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("heads, lengths", [(2, [70, 130]), (16, [70, 64, 1, 131, 33])], ids=["few chains", "many chains"])
def test_delta_rule_into_rows_that_begin_anywhere(dtype, heads, lengths):
    """`out` needs a contiguous last dimension and no alignment; what lies around it stays."""
    x = gpu(make(lengths, heads, heads, 64, 64, TYPES[dtype], True, seed=41))
    n = sum(lengths)
    kw = dict(initial_state=x["initial"], offsets=torch.tensor(ends(lengths), dtype=torch.int32, device="cuda"))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    want = ops.delta_rule(*args, **kw)
    step = ops.delta_rule_step(*(t[:7] for t in args), torch.zeros(7, heads, 64, 64, device="cuda"))
    for lead in (1, 3):
        around = torch.full((n, heads, 64 + 2 * lead + 1), 5.0, device="cuda", dtype=TYPES[dtype])
        o, s = ops.delta_rule(*args, out=around[:, :, lead:lead + 64], **kw)
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])
        assert bool((around[:, :, :lead] == 5).all()) and bool((around[:, :, lead + 64:] == 5).all())
        o = ops.delta_rule_step(*(t[:7] for t in args), torch.zeros(7, heads, 64, 64, device="cuda"), out=around[:7, :, lead:lead + 64])
        assert torch.equal(o, step) and bool((around[:, :, :lead] == 5).all()) and bool((around[:, :, lead + 64:] == 5).all())


@pytest.mark.gpu
def test_delta_rule_captured_once_and_replayed_with_other_lengths():
    """Offsets on the GPU are read when the kernels run: a graph takes whatever lengths are in them at a replay."""
    x = gpu(make([200], 2, 4, 64, 64, torch.bfloat16, False, seed=43))
    first = torch.randn(3, 4, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    off = torch.tensor([0, 70, 130, 200], dtype=torch.int32, device="cuda")
    args, kw = (x["q"], x["k"], x["v"], x["g"], x["beta"]), dict(initial_state=first, offsets=off)

    def work():
        o, s, saved = ops.delta_rule(*args, keep=True, **kw)
        return (o, s) + ops.delta_rule_backward(x["do"], *args, saved=saved, **kw)
    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for at in ([0, 70, 130, 200], [0, 0, 1, 64], [0, 128, 128, 199], [0, 0, 0, 0], [0, 0, 0, 200], [0, 70, 130, 200]):
        off.copy_(torch.tensor(at, dtype=torch.int32))
        want = work()
        for t in got:
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), at
        assert not got[0][at[-1]:].any() and not got[2][at[-1]:].any()


@pytest.mark.gpu
def test_delta_rule_of_tokens_in_no_sequence():
    x = gpu(make([10], 1, 2, 64, 64, torch.float32, False, seed=47))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    first = torch.randn(2, 2, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    for off in ([0, 0, 0], torch.zeros(3, dtype=torch.int64, device="cuda")):
        o, s, saved = ops.delta_rule(*args, initial_state=first, offsets=off, keep=True)
        assert not o.any() and torch.equal(s, first)
        got = ops.delta_rule_backward(x["do"], *args, initial_state=first, offsets=off, d_final_state=first, saved=saved)
        assert not any(t.any() for t in got[:5]) and torch.equal(got[5], first)


@pytest.mark.gpu
def test_delta_rule_with_a_state_that_grows():
    """Positive g, as long as e to their sum over 64 tokens is a float32: of 64 tokens two thirds have up to 0.3."""
    lengths = [64, 40]
    x = make(lengths, 1, 2, 64, 64, torch.float32, True, seed=53)
    x["g"] = x["g"].abs().clamp(max=0.3)
    x["g"][::3] *= -1.0
    check_delta(x, lengths)


@pytest.mark.gpu
def test_delta_rule_backward_keeps_a_nan_in_its_sequence_and_head():
    lengths = [70, 80]
    d = gpu(make(lengths, 2, 2, 64, 64, torch.bfloat16, False, seed=59))
    off = torch.tensor(ends(lengths), dtype=torch.int32, device="cuda")
    names = ("q", "k", "v", "g", "beta")
    want = ops.delta_rule_backward(d["do"], *(d[n] for n in names), offsets=off)
    for where in ("v", "do"):
        spoiled = dict(d)
        spoiled[where] = d[where].clone()
        spoiled[where][66, 1, 3] = math.nan
        got = ops.delta_rule_backward(spoiled["do"], *(spoiled[n] for n in names), offsets=off)
        for a, b in zip(got[:5], want):
            assert torch.equal(a[:, 0], b[:, 0]) and torch.equal(a[70:], b[70:])
        assert torch.equal(got[5][1], want[5][1]) and torch.equal(got[5][0, 0], want[5][0, 0])
        assert bool(got[1][:70, 1].isnan().any())


@pytest.mark.gpu
def test_delta_step_over_an_empty_pool_and_padded_rows_alone():
    x = gpu(make([5], 1, 2, 64, 64, torch.bfloat16, False, seed=61))
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    slots = torch.full((5,), -1, dtype=torch.int32, device="cuda")
    assert not ops.delta_rule_step(*args, torch.zeros(0, 2, 64, 64, device="cuda"), slots=slots).any()
    state = torch.randn(3, 2, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    kept = state.clone()
    assert not ops.delta_rule_step(*args, state, slots=slots).any() and torch.equal(state, kept)
    slots[2] = 0
    o = ops.delta_rule_step(*args, torch.zeros(0, 2, 64, 64, device="cuda"), slots=slots)
    assert bool(o[2].isnan().all()) and not o[[0, 1, 3, 4]].any()


@pytest.mark.gpu
def test_layer_norm_autograd_with_a_bias_alone_and_a_broadcast_gradient():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 5, 40, generator=gen).bfloat16().cuda()
    for kind in (torch.bfloat16, torch.float32):
        leaf, b = x.clone().requires_grad_(), torch.randn(40, generator=gen).to(kind).cuda().requires_grad_()
        ops.LayerNorm.apply(leaf, None, b).sum().backward()
        assert b.grad.dtype == kind and bool((b.grad == 30).all())
        # a sum over the row of what has no mean: zero up to the rounding of dy and of the two means
        assert leaf.grad.shape == x.shape and float(leaf.grad.float().abs().max()) <= 8 * 40 * U * float(1 / x.float().std(-1, correction=0).min())
    w = torch.ones(40, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.ones(40, device="cuda", dtype=torch.bfloat16).expand(6, 5, 40)
    y = ops.LayerNorm.apply(x, w)
    y.backward(dy)
    _, mean, rstd = ops.layer_norm(x)
    assert torch.equal(w.grad, ops.layer_norm_backward(dy.contiguous(), x, w.detach(), mean, rstd)[1])


@pytest.mark.gpu
def test_c_entries_without_what_may_be_null():
    """No initial, final or d_final state, no gradient of the initial one, no statistics and no gradient of the weight or the bias."""
    x = gpu(make([130], 1, 2, 64, 64, torch.float32, False, seed=67))
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    args = (x["q"], x["k"], x["v"], x["g"], x["beta"])
    o, s, saved = ops.delta_rule(*args, scale=0.5, keep=True)
    want = ops.delta_rule_backward(x["do"], *args, scale=0.5, saved=saved)
    c = _lib.HelenDeltaRuleC()
    c.struct_size, c.device, c.dtype = ctypes.sizeof(c), x["q"].get_device(), _lib.HELEN_TYPE_FP32
    c.heads_k, c.heads_v, c.width_k, c.width_v, c.tokens, c.sequences, c.scale = 1, 2, 64, 64, 130, 1, 0.5
    pair = lambda t: (ctypes.c_int64 * 2)(*t.stride()[:2])  # noqa: E731
    for name, t in zip(("q", "k", "v", "g", "beta", "d_o"), args + (x["do"],)):
        setattr(c, name, t.data_ptr())
        setattr(c, name + "_stride", pair(t))
    sizes = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(lib.helen_delta_rule_bytes(ctypes.byref(c), *(ctypes.byref(t) for t in sizes)))
    kept, own = (torch.empty(t.value, dtype=torch.uint8, device="cuda") for t in sizes[1:])
    out, state = torch.full_like(o, 7.0), torch.full_like(s, 7.0)
    got = [torch.full_like(t, 7.0) for t in want[:5]]
    for name, t in zip(("grad_q", "grad_k", "grad_v", "grad_g", "grad_beta"), got):
        setattr(c, name, t.data_ptr())
    c.final_state = state.data_ptr()                      # the states alone
    _lib.check(lib.helen_delta_rule_forward(ctypes.byref(c), 1, kept.data_ptr(), kept.numel(), stream))
    assert torch.equal(state, s)
    c.o, c.o_stride, c.final_state = out.data_ptr(), pair(out), None      # the outputs alone
    _lib.check(lib.helen_delta_rule_forward(ctypes.byref(c), 1, kept.data_ptr(), kept.numel(), stream))
    _lib.check(lib.helen_delta_rule_backward(ctypes.byref(c), kept.data_ptr(), kept.numel(), own.data_ptr(), own.numel(), stream))
    assert torch.equal(out, o) and all(torch.equal(a, b) for a, b in zip(got, want))
    rows, width = 300, 100
    gen = torch.Generator().manual_seed(5)
    y, dy, w = (torch.randn(*shape, generator=gen).cuda() for shape in ((rows, width), (rows, width), (width,)))
    norm, mean, rstd = ops.layer_norm(y, w, w)
    dx, dw, db = ops.layer_norm_backward(dy, y, w, mean, rstd)
    n = _lib.HelenLayerNormC()
    n.struct_size, n.device, n.width, n.rows, n.eps = ctypes.sizeof(n), y.get_device(), width, rows, 1e-5
    n.x, n.x_stride, n.weight, n.bias = y.data_ptr(), width, w.data_ptr(), w.data_ptr()
    out, grad, sums = torch.empty_like(y), torch.empty_like(y), torch.full((2, width), 7.0, device="cuda")
    n.y, n.y_stride = out.data_ptr(), width
    _lib.check(lib.helen_layer_norm_forward(ctypes.byref(n), stream))
    assert torch.equal(out, norm)
    n.mean, n.rstd, n.dy, n.dy_stride, n.dx, n.dx_stride = mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), width, grad.data_ptr(), width
    need = ctypes.c_size_t()
    _lib.check(lib.helen_layer_norm_bytes(ctypes.byref(n), ctypes.byref(need)))
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    for a, b in ((None, None), (sums[0], None), (None, sums[1])):
        grad.fill_(7.0)
        sums.fill_(7.0)
        n.dweight, n.dbias = (None if t is None else t.data_ptr() for t in (a, b))
        _lib.check(lib.helen_layer_norm_backward(ctypes.byref(n), work.data_ptr(), work.numel(), stream))
        assert torch.equal(grad, dx)
        assert torch.equal(sums[0], torch.full_like(dw, 7.0) if a is None else dw)
        assert torch.equal(sums[1], torch.full_like(db, 7.0) if b is None else db)
