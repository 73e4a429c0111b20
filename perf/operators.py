"""The sequence operators and what their speed is measured on: the gated delta rule over whole sequences (forward, and
forward with backward), its single-token form over a pool of states, and layer norm (forward, and forward with backward).

`own` False computes the plain forms (elementary torch operations in 32 bits), `own` True calls helen_amd.sequence_ops.

The gated delta rule keeps per value head a state S [Dk, Dv] and takes a token (q, k in R^Dk, v in R^Dv, log decay g,
step beta) as

    u = beta (v - e^g S^T k),    S <- e^g S + k u^T,    o = scale S^T q

with Hk query / key heads shared by Hv value heads.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CHUNK = 64


# ---------------------------------------------------------------------------------------------------------------- cases
def _delta(kind, name, dtype, heads_k, heads_v, dk, dv, lengths, initial):
    return {"kind": kind, "name": name, "dtype": dtype, "heads_k": heads_k, "heads_v": heads_v, "dk": dk, "dv": dv,
            "lengths": lengths, "initial": initial}


def _step(name, dtype, rows, live, pool, heads_k, heads_v, dk, dv):
    return {"kind": "step", "name": name, "dtype": dtype, "rows": rows, "live": live, "pool": pool, "heads_k": heads_k,
            "heads_v": heads_v, "dk": dk, "dv": dv}


def _norm(kind, name, dtype, rows, width, weight):
    return {"kind": kind, "name": name, "dtype": dtype, "rows": rows, "width": width, "weight": weight}


def listed():
    return [
        # one generated token of one stream: what counts is the latency of the call
        _step("step: one stream", "bf16", 1, 1, 4, 4, 8, 128, 128),
        # a serving batch padded to a fixed size (four rows behind the last stream), its streams anywhere in the pool
        _step("step: 256 streams", "bf16", 256, 252, 384, 16, 32, 128, 128),
        # an odd batch of the smaller state, everything in fp32
        _step("step: 37 streams fp32", "fp32", 37, 37, 48, 4, 8, 64, 64),
        # one chunk of a pileup window (100 positions) in fp32: the smallest whole-sequence call
        _delta("forward", "forward: 100 tokens fp32", "fp32", 2, 2, 128, 128, "100", False),
        # 64 pileup windows of 1000 positions, hidden width 4 x 128
        _delta("forward", "forward: 64 windows", "bf16", 4, 4, 128, 128, "64x1000", False),
        # one long prompt: few chains, each long
        _delta("forward", "forward: 16384 tokens", "bf16", 16, 32, 128, 128, "16384", True),
        # prompts of different lengths packed behind one another, going on from their states, in half precision
        _delta("forward", "forward: ragged fp16", "fp16", 4, 16, 64, 128, "1,63,64,65,100,1000,2777,517,0,1900", True),
        # a training step's two passes over 32 windows
        _delta("train", "train: 32 windows", "bf16", 4, 8, 128, 128, "32x1000", False),
        # a training step's two passes over two packed documents, going on from a state
        _delta("train", "train: 8191 tokens", "bf16", 8, 16, 128, 128, "5000,3191", True),
        # the norm of one chunk's positions (100 x 128): latency
        _norm("norm", "norm: 100 x 128", "fp32", 100, 128, "fp32"),
        # the norm of the heads' outputs of a long prompt
        _norm("norm", "norm: 262143 x 128", "bf16", 262143, 128, "bf16"),
        # a training step's two passes of the norm over the hidden width
        _norm("norm_train", "norm train: 32000 x 2048", "bf16", 32000, 2048, "fp32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["step", "forward", "forward", "train", "train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("norm", "norm_train"):
        width = _spread(rng, 64, 4096)
        rows = _spread(rng, 16, max(17, 33_000_000 // width))
        return {"kind": kind, "dtype": dtype, "rows": rows, "width": width, "weight": rng.choice(["fp32", dtype])}
    heads_k = rng.choice([1, 2, 3, 4, 8, 16])
    heads_v = heads_k * rng.choice([1, 2, 3])
    dk, dv = rng.choice([64, 128]), rng.choice([64, 128])
    if kind == "step":
        rows = _spread(rng, 1, max(2, 8000 // heads_v))
        live = rows - rng.choice([0, 0, rows // 8])
        return {"kind": kind, "dtype": dtype, "rows": rows, "live": live, "pool": rows + rng.randrange(0, rows + 1),
                "heads_k": heads_k, "heads_v": heads_v, "dk": dk, "dv": dv}
    most = min(16000, (400_000 if kind == "forward" else 110_000) // heads_v)
    if dtype == "fp32":
        most //= 2
    total = _spread(rng, 64, most)
    sequences = min(total, _spread(rng, 1, 40))
    cuts = sorted(rng.randrange(0, total + 1) for _ in range(sequences - 1))
    ends = [0] + cuts + [total]
    lengths = ",".join(str(b - a) for a, b in zip(ends, ends[1:]))
    return {"kind": kind, "dtype": dtype, "heads_k": heads_k, "heads_v": heads_v, "dk": dk, "dv": dv,
            "lengths": lengths, "initial": rng.random() < 0.5}


def _lengths(case):
    got = []
    for part in case["lengths"].split(","):
        n, _, each = part.partition("x")
        got += [int(each)] * int(n) if each else [int(n)]
    return got


# --------------------------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _unit(x):
    return x / x.square().sum(-1, keepdim=True).add(1e-6).sqrt()


def _tokens(gen, n, case):
    """q, k of length one, v, log decays from slow to fast ones per head, steps in (0, 1): what a layer's projections and
    gates give."""
    t = _TYPES[case["dtype"]]
    hk, hv, dk, dv = case["heads_k"], case["heads_v"], case["dk"], case["dv"]
    rate = torch.linspace(-5.0, 0.5, hv, device="cuda").exp() if hv > 1 else torch.full((1,), 0.05, device="cuda")
    return {"q": _unit(_normal(gen, n, hk, dk)).to(t), "k": _unit(_normal(gen, n, hk, dk)).to(t),
            "v": _normal(gen, n, hv, dv).to(t),
            "g": -rate * torch.nn.functional.softplus(_normal(gen, n, hv)),
            "beta": torch.sigmoid(_normal(gen, n, hv)), "scale": dk ** -0.5}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    t = _TYPES[case["dtype"]]
    s = {"kind": kind}
    if kind in ("norm", "norm_train"):
        rows, width, w = case["rows"], case["width"], _TYPES[case["weight"]]
        s["x"] = (_normal(gen, rows, width) * 1.5 + 0.3 * _normal(gen, rows, 1)).to(t)
        s["weight"] = (1.0 + 0.2 * _normal(gen, width)).to(w)
        s["bias"] = (0.2 * _normal(gen, width)).to(w)
        if kind == "norm_train":
            s["dy"] = _normal(gen, rows, width).to(t)
        return s
    if kind == "step":
        s.update(_tokens(gen, case["rows"], case))
        shape = (case["pool"], case["heads_v"], case["dk"], case["dv"])
        s["state"] = _normal(gen, *shape) * 0.3
        order = torch.randperm(case["pool"], generator=gen, device="cuda")[:case["rows"]].to(torch.int32)
        order[case["live"]:] = -1
        s["slots"], s["live"] = order.contiguous(), case["live"]
        return s
    lengths = _lengths(case)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    s.update(_tokens(gen, ends[-1], case))
    s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    s["longest"] = max(lengths)
    shape = (len(lengths), case["heads_v"], case["dk"], case["dv"])
    s["initial"] = _normal(gen, *shape) * 0.3 if case["initial"] else None
    if kind == "train":
        s["do"] = _normal(gen, ends[-1], case["heads_v"], case["dv"]).to(t)
        s["d_final"] = _normal(gen, *shape) * 0.3 if case["initial"] else None
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _padded_rows(s):
    """Token index of every position of the sequences, padded to whole chunks, and which of them are tokens."""
    off = s["offsets"].long()
    pad = -(-max(s["longest"], 1) // _CHUNK) * _CHUNK
    at = off[:-1, None] + torch.arange(pad, device=off.device)[None]
    live = at < off[1:, None]
    return at.clamp(max=max(int(s["q"].shape[0]) - 1, 0)), live


def _plain_chunks(q, k, v, g, beta, scale, state):
    """The delta rule in chunks, everything [sequence, head, chunk, 64, ...] in fp32; positions that are no tokens have
    k = 0, beta = 0 and g = 0.  The log decays between two positions are differences of sums in 64 bits."""
    total = g.double().cumsum(-1)
    between = total[..., :, None] - total[..., None, :]
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = between.masked_fill(~lower, -math.inf).exp().float()
    from_start, to_end = total.exp().float()[..., None], (total[..., -1:] - total).exp().float()[..., None]
    whole = total[..., -1].exp().float()[..., None, None]
    kt = k.transpose(-1, -2)
    system = -(beta[..., None] * (k @ kt) * decay).masked_fill(~lower.tril(-1), 0.0)
    inverse, power = torch.eye(_CHUNK, device=q.device) + system, system
    for _ in range(5):   # (I - N)^-1 = (I + N)(I + N^2)(I + N^4)...: N is strictly lower, N^64 = 0
        power = power @ power
        inverse = inverse + inverse @ power
    scores = (q @ kt) * decay
    new_v = inverse @ (beta[..., None] * v)
    new_k = inverse @ (beta[..., None] * from_start * k)
    q_in, k_out = q * from_start, (k * to_end).transpose(-1, -2)
    o = []
    for c in range(q.shape[2]):
        u = new_v[:, :, c] - new_k[:, :, c] @ state
        o.append(scale * (q_in[:, :, c] @ state + scores[:, :, c] @ u))
        state = whole[:, :, c] * state + k_out[:, :, c] @ u
    return torch.stack(o, 2), state


def _plain_delta(s):
    train = s["kind"] == "train"
    tokens, hv, dv = s["v"].shape
    hk, dk = s["q"].shape[1:]
    if tokens == 0:
        raise ValueError("no tokens")
    at, live = _padded_rows(s)
    n, pad = at.shape
    mask = live[:, :, None, None]
    first = s["initial"] if s["initial"] is not None else torch.zeros(n, hv, dk, dv, device=at.device)
    leaves = [s["q"].float(), s["k"].float(), s["v"].float(), s["g"], s["beta"], first]
    if train:
        leaves = [x.detach().clone().requires_grad_() for x in leaves]

    def chunks(x, per):
        x = torch.where(mask, x[at], x.new_zeros(()))
        x = x[:, :, :, None].expand(-1, -1, -1, per, -1).reshape(n, pad // _CHUNK, _CHUNK, hv, x.shape[-1])
        return x.permute(0, 3, 1, 2, 4)

    with torch.set_grad_enabled(train):
        q, k, v, g, beta, first = leaves
        o, last = _plain_chunks(chunks(q, hv // hk), chunks(k, hv // hk), chunks(v, 1), chunks(g[..., None], 1)[..., 0],
                                chunks(beta[..., None], 1)[..., 0], s["scale"], first)
        o = o.permute(0, 2, 3, 1, 4).reshape(n * pad, hv, dv)
        back = torch.zeros(tokens, dtype=torch.long, device=at.device)
        place = torch.arange(n * pad, device=at.device)
        back = back.index_add(0, at.reshape(-1), torch.where(live.reshape(-1), place, place.new_zeros(())))
        o = o[back]
        if not train:
            return {"o": o.to(s["v"].dtype), "state": last}
        outs, seeds = [o], [s["do"].float()]
        if s["d_final"] is not None:
            outs, seeds = outs + [last], seeds + [s["d_final"]]
        dq, dk_, dv_, dg, dbeta, dfirst = torch.autograd.grad(outs, leaves, seeds)
    t = s["v"].dtype
    got = {"o": o.detach().to(t), "state": last.detach(), "dq": dq.to(t), "dk": dk_.to(t), "dv": dv_.to(t), "dg": dg,
           "dbeta": dbeta}
    if s["initial"] is not None:
        got["d_initial"] = dfirst
    return got


def _plain_step(s):
    n, group = s["live"], s["v"].shape[1] // s["q"].shape[1]
    at = s["slots"][:n].long()
    q = s["q"][:n].float().repeat_interleave(group, 1)
    k = s["k"][:n].float().repeat_interleave(group, 1)
    state = s["state"][at] * s["g"][:n].exp()[..., None, None]
    u = s["beta"][:n, :, None] * (s["v"][:n].float() - (state * k[..., None]).sum(-2))
    state = state + k[..., None] * u[..., None, :]
    s["state"].index_copy_(0, at, state)
    o = torch.zeros_like(s["v"])
    o[:n] = (s["scale"] * (state * q[..., None]).sum(-2)).to(o.dtype)
    return {"o": o, "state": s["state"]}


def _plain_norm(s, eps=1e-5):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(-1, keepdim=True)
    away = x - mean
    rstd = (away.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = away * rstd
    t, wt = s["x"].dtype, s["weight"].dtype
    got = {"y": (unit * w + b).to(t), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if s["kind"] == "norm_train":
        dy = s["dy"].float()
        dunit = dy * w
        dx = rstd * (dunit - dunit.mean(-1, keepdim=True) - unit * (dunit * unit).mean(-1, keepdim=True))
        got.update(dx=dx.to(t), dweight=(dy * unit).sum(0).to(wt), dbias=dy.sum(0).to(wt))
    return got


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    s, kind = state, state["kind"]
    if own:
        from helen_amd import sequence_ops as ops
        if kind in ("norm", "norm_train"):
            y, mean, rstd = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
            got = {"y": y, "mean": mean, "rstd": rstd}
            if kind == "norm_train":
                got["dx"], got["dweight"], got["dbias"] = ops.layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd)
            return got
        if kind == "step":
            o = ops.delta_rule_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], slots=s["slots"],
                                    scale=s["scale"])
            return {"o": o, "state": s["state"]}
        if kind == "forward":
            o, last = ops.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"],
                                     initial_state=s["initial"], offsets=s["offsets"])
            return {"o": o, "state": last}
        o, last, saved = ops.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"],
                                        initial_state=s["initial"], offsets=s["offsets"], keep=True)
        dq, dk, dv, dg, dbeta, dfirst = ops.delta_rule_backward(
            s["do"], s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"], initial_state=s["initial"],
            offsets=s["offsets"], d_final_state=s["d_final"], saved=saved)
        got = {"o": o, "state": last, "dq": dq, "dk": dk, "dv": dv, "dg": dg, "dbeta": dbeta}
        if s["initial"] is not None:
            got["d_initial"] = dfirst
        return got
    return _plain_norm(s) if kind in ("norm", "norm_train") else _plain_step(s) if kind == "step" else _plain_delta(s)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        n = case["rows"] * case["width"]
        w = {"bf16": 2, "fp16": 2, "fp32": 4}[case["weight"]]
        passes = 2 if kind == "norm" else 4          # x, y; and dy, dx (x stays in reach only where it is small)
        return {"bytes": passes * n * size + (2 if kind == "norm" else 4) * w * case["width"] + 8 * case["rows"],
                "flops": (8 if kind == "norm" else 20) * n}
    hk, hv, dk, dv = case["heads_k"], case["heads_v"], case["dk"], case["dv"]
    per_token = 2 * hk * dk * size + hv * dv * size + 2 * hv * 4
    if kind == "step":
        n = case["live"]
        return {"bytes": n * (per_token + hv * dv * size + 2 * 4 * hv * dk * dv), "flops": n * hv * 7 * dk * dv}
    lengths = _lengths(case)
    n, states = sum(lengths), len(lengths) * hv * dk * dv * 4
    moved = n * (per_token + hv * dv * size) + states * (2 if case["initial"] else 1)
    flops = n * hv * 6 * dk * dv
    if kind == "train":
        moved += n * (per_token + hv * dv * size) + n * per_token + states * (3 if case["initial"] else 0)
        flops += n * hv * 14 * dk * dv
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_delta(s):
    """Token by token in 64 bits, by the recurrence; the gradients by its reverse, over states kept every 32 tokens."""
    d = torch.float64
    n, hv = s["offsets"].numel() - 1, s["v"].shape[1]
    group = hv // s["q"].shape[1]
    dk, dv = s["q"].shape[2], s["v"].shape[2]
    off = [int(x) for x in s["offsets"].tolist()]
    longest, dev = s["longest"], s["q"].device
    order = sorted(range(n), key=lambda i: off[i] - off[i + 1])       # the longest first: a step takes the first m of them
    count = [off[i + 1] - off[i] for i in order]
    start = torch.tensor([off[i] for i in order], device=dev)
    index = torch.tensor(order, device=dev)
    m_at, m = [], n
    for t in range(longest):
        while m and count[m - 1] <= t:
            m -= 1
        m_at.append(m)

    def token(t):
        r = start[:m_at[t]] + t
        wide = lambda x: x[r].to(d).repeat_interleave(group, 1)  # noqa: E731
        return r, wide(s["q"]), wide(s["k"]), s["v"][r].to(d), s["g"][r].to(d).exp()[..., None, None], s["beta"][r].to(d)[..., None]

    def mv(mat, vec):        # vec^T mat
        return torch.matmul(vec.unsqueeze(-2), mat).squeeze(-2)

    def step(S, t):
        r, q, k, v, a, beta = token(t)
        m = m_at[t]
        aS = S[:m] * a
        miss = v - mv(aS, k)
        new = aS + k.unsqueeze(-1) * (beta * miss).unsqueeze(-2)
        return r, q, k, v, a, beta, aS, miss, new

    S = torch.zeros(n, hv, dk, dv, dtype=d, device=dev)
    if s["initial"] is not None:
        S += s["initial"].to(d)[index]
    o = torch.zeros(s["v"].shape, dtype=d, device=dev)
    train, every, kept = s["kind"] == "train", 32, []
    for t in range(longest):
        if train and t % every == 0:
            kept.append(S.clone())
        r, q, k, v, a, beta, aS, miss, new = step(S, t)
        S[:m_at[t]] = new
        o[r] = s["scale"] * mv(new, q)
    last = torch.empty_like(S)
    last[index] = S
    got = {"o": o, "state": last}
    if not train:
        return got
    G = torch.zeros_like(S)
    if s["d_final"] is not None:
        G += s["d_final"].to(d)[index]
    dq, dk_ = (torch.zeros(s["v"].shape[0], hv, dk, dtype=d, device=dev) for _ in range(2))
    dv_ = torch.zeros(s["v"].shape, dtype=d, device=dev)
    dg, dbeta = (torch.zeros(s["g"].shape, dtype=d, device=dev) for _ in range(2))
    for block in reversed(range(len(kept))):
        S, low = kept[block], block * every
        path = []
        for t in range(low, min(longest, low + every)):
            path.append(S)
            new = step(S, t)[-1]
            S = S.clone()
            S[:m_at[t]] = new
        kept[block] = None
        for t in reversed(range(low, min(longest, low + every))):
            m = m_at[t]
            r, q, k, v, a, beta, aS, miss, new = step(path.pop(), t)
            do = s["do"][r].to(d) * s["scale"]
            dq[r] = torch.matmul(new, do.unsqueeze(-1)).squeeze(-1)
            D = G[:m] + q.unsqueeze(-1) * do.unsqueeze(-2)
            du = mv(D, k)
            dbeta[r] = (du * miss).sum(-1)
            dmiss = beta * du
            dv_[r] = dmiss
            dk_[r] = torch.matmul(D, (beta * miss).unsqueeze(-1)).squeeze(-1) - torch.matmul(aS, dmiss.unsqueeze(-1)).squeeze(-1)
            D = D - k.unsqueeze(-1) * dmiss.unsqueeze(-2)
            dg[r] = (D * aS).sum((-1, -2))
            G[:m] = a * D
    share = lambda x: x.view(x.shape[0], -1, group, dk).sum(2)  # noqa: E731
    got.update(dq=share(dq), dk=share(dk_), dv=dv_, dg=dg, dbeta=dbeta)
    if s["initial"] is not None:
        first = torch.empty_like(G)
        first[index] = G
        got["d_initial"] = first
    return got


def _exact_step(s):
    d = torch.float64
    o, state = torch.zeros(s["v"].shape, dtype=d, device="cuda"), s["state"].to(d)
    group = s["v"].shape[1] // s["q"].shape[1]
    for row, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            q, k = (s[x][row].to(d).repeat_interleave(group, 0) for x in ("q", "k"))
            S = state[slot] * s["g"][row].to(d).exp()[:, None, None]
            miss = s["v"][row].to(d) - torch.matmul(k.unsqueeze(-2), S).squeeze(-2)
            S = S + k.unsqueeze(-1) * (s["beta"][row].to(d)[:, None] * miss).unsqueeze(-2)
            state[slot] = S
            o[row] = s["scale"] * torch.matmul(q.unsqueeze(-2), S).squeeze(-2)
    return {"o": o, "state": state}


def _exact_norm(s, eps=1e-5):
    x, w = s["x"].double(), s["weight"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    got = {"y": (x - mean) * rstd * w + s["bias"].double(), "mean": mean.flatten(), "rstd": rstd.flatten()}
    if s["kind"] == "norm_train":
        h, dy = (x - mean) * rstd, s["dy"].double()
        e = dy * w
        n = x.shape[1]
        got["dx"] = rstd / n * (n * e - e.sum(1, keepdim=True) - h * (e * h).sum(1, keepdim=True))
        got["dweight"], got["dbias"] = torch.einsum("ij,ij->j", dy, h), dy.sum(0)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    return _exact_norm(s) if kind in ("norm", "norm_train") else _exact_step(s) if kind == "step" else _exact_delta(s)
