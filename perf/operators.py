"""Cases that time and check the gated delta rule and the 8-bit activation checkpoints.

Six operators of ``fpscan_b200``:

* ``prefill`` -- ``gated_delta_forward``: the gated delta rule over a sequence, entering with a state and
  returning the last one (what a server does with a prompt);
* ``train``   -- ``gated_delta`` and the gradients of all its inputs;
* ``train8``  -- the same with ``checkpoint8=True``: q, k and v are kept for the backward pass in 8 bits;
* ``step``    -- ``gated_delta_step``: one or a few tokens per sequence, the state updated in place;
* ``scan8``   -- ``pscan_channels_last(..., checkpoint8=True)`` and its gradients: the output is kept for the
  backward pass in 8 bits;
* ``round8``  -- ``quantize8`` and ``dequantize8``: the checkpoint itself, written and read back.

The rule, for one head with a state S of (Dv, Dk), a = exp(log_decay):

    S_t = a_t S_{t-1} + beta_t (v_t - a_t S_{t-1} k_t) k_t^T,      o_t = scale S_t q_t.

With ``own`` false ``run`` computes this in chunks of elementary torch operations in 32 bits (the decays and the
small triangular inverse in 64); with ``own`` true it makes the calls that a user makes.
"""
import math

import torch

own = False

CHUNK = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FLOOR = -150.0  # exp(-150) is 0 in 32 bits: stands for a log_decay of -inf (a reset)


# ------------------------------------------------------------------------------------------------ cases
def _delta(name, op, batch, seqlen, key_heads, group, dk, dv, dtype, state=False, resets=False):
    case = {"op": op, "batch": batch, "seqlen": seqlen, "key_heads": key_heads, "group": group,
            "dk": dk, "dv": dv, "dtype": dtype, "state": state, "resets": resets}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one sequence of a small model, one token: the latency of a call
        _delta("step, one sequence", "step", 1, 1, 4, 1, 64, 64, "bf16"),
        # a server's batch, one token each, two value heads to a key head: the states' bytes
        _delta("step, a batch of 256", "step", 256, 1, 16, 2, 128, 128, "bf16"),
        # short prompts of a ragged length, heads of odd sizes, documents packed behind each other
        _delta("prefill, short and ragged", "prefill", 3, 333, 2, 3, 64, 96, "fp16", state=True, resets=True),
        # two long prompts
        _delta("prefill, two of 8192", "prefill", 2, 8192, 8, 2, 128, 128, "bf16", state=True),
        # a numerics run in full precision, with a learned initial state
        _delta("train, small fp32", "train", 2, 200, 4, 1, 64, 64, "fp32", state=True),
        # a training step's layer
        _delta("train, 4 of 4096", "train", 4, 4096, 16, 1, 128, 128, "bf16"),
        # a fine-tuning batch of one ragged sequence, checkpoints in 8 bits
        _delta("train8, one of 777", "train8", 1, 777, 4, 2, 96, 64, "fp16"),
        # a training step's layer with shared key heads, checkpoints in 8 bits
        _delta("train8, 2 of 2048", "train8", 2, 2048, 8, 2, 128, 128, "bf16"),
        # a narrow layer over one long sequence: few columns, cut along the time axis
        {"name": "scan8, narrow", "op": "scan8", "batch": 1, "seqlen": 5000, "dim": 512, "dtype": "fp16"},
        # the channel-last benchmark's bf16 layer
        {"name": "scan8, 8 x 8192 x 2048", "op": "scan8", "batch": 8, "seqlen": 8192, "dim": 2048, "dtype": "bf16"},
        # a small activation of an odd size
        {"name": "round8, small", "op": "round8", "rows": 77, "dim": 1001, "dtype": "bf16"},
        # a layer's hidden states
        {"name": "round8, 32768 x 4096", "op": "round8", "rows": 32768, "dim": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "train", "train", "train8", "step", "step", "scan8", "round8"])
    if op == "scan8":
        return {"op": op, "batch": _log(rng, 1, 8), "seqlen": _log(rng, 1, 8192), "dim": 8 * _log(rng, 4, 256),
                "dtype": rng.choice(["bf16", "fp16"])}
    if op == "round8":
        return {"op": op, "rows": _log(rng, 1, 32768), "dim": _log(rng, 1, 4096), "dtype": rng.choice(sorted(TYPES))}
    dk, dv = rng.choice([16, 32, 40, 64, 64, 96, 128, 128]), rng.choice([16, 32, 64, 72, 96, 128, 128, 192])
    key_heads, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 3])
    if op == "step":
        batch, seqlen = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 3, 5, 8])
        key_heads, dv = min(key_heads, 10), min(dv, 128)
        return _delta("", op, batch, seqlen, key_heads, group, dk, dv, rng.choice(sorted(TYPES)), resets=rng.random() < 0.2)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"] if op != "train8" else ["bf16", "fp16"])
    seqlen = _log(rng, 1, 8192 if op == "prefill" else 4096)
    most = (1 << 17) // (seqlen * key_heads * group) + 1  # half of the largest listed case's heads x tokens
    return _delta("", op, min(_log(rng, 1, 8), most), seqlen, key_heads, group, dk, dv, dtype,
                  state=op == "prefill" or (op == "train" and rng.random() < 0.3), resets=rng.random() < 0.25)


# ------------------------------------------------------------------------------------------------ inputs
def _make_delta(case, gen):
    t = TYPES[case["dtype"]]
    b, l, hk, dk, dv = (case[n] for n in ("batch", "seqlen", "key_heads", "dk", "dv"))
    h = hk * case["group"]
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    # keys and queries of unit length, write strengths in (0, 1), decays of a selective layer: most close to 1
    s = {"q": unit(rand(b, l, hk, dk)).to(t), "k": unit(rand(b, l, hk, dk)).to(t), "v": rand(b, l, h, dv).to(t),
         "beta": torch.sigmoid(rand(b, l, h)).to(t)}
    rate = torch.exp(rand(h) - 1.0)
    g = -rate * torch.nn.functional.softplus(rand(b, l, h) - 1.0)
    if case["resets"]:  # a document begins: the state before it counts no more
        g = torch.where(torch.rand(b, l, h, generator=gen, device="cuda") < 0.01, -math.inf, g)
    s["log_decay"] = g.to(t)
    s["scale"] = dk ** -0.5
    return s, rand


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "scan8":
        t, shape = TYPES[case["dtype"]], (case["batch"], case["seqlen"], case["dim"])
        z = torch.randn(shape, generator=gen, device="cuda")
        return {"op": op, "gates": torch.sigmoid(z + 2.0).to(t).requires_grad_(),
                "tokens": torch.randn(shape, generator=gen, device="cuda").to(t).requires_grad_(),
                "grad": torch.randn(shape, generator=gen, device="cuda").to(t)}
    if op == "round8":
        x = torch.randn(case["rows"], case["dim"], generator=gen, device="cuda")
        return {"op": op, "x": (x * torch.exp(torch.randn(case["rows"], 1, generator=gen, device="cuda"))).to(TYPES[case["dtype"]])}
    s, rand = _make_delta(case, gen)
    b, h, dk, dv = case["batch"], case["key_heads"] * case["group"], case["dk"], case["dv"]
    s["op"] = op
    if op == "step" or case["state"]:
        s["state"] = rand(b, h, dv, dk) * 0.1
    if op in ("train", "train8"):
        for n in LEAVES + (("state",) if case["state"] else ()):
            s[n].requires_grad_()
        s["grad"] = rand(b, case["seqlen"], h, dv).to(s["v"].dtype)
        if case["state"]:
            s["grad_state"] = rand(b, h, dv, dk) * 0.1
    return s


LEAVES = ("q", "k", "v", "log_decay", "beta")


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_delta(q, k, v, log_decay, beta, state, scale):
    """The rule in chunks, 32 bits: the rank-C update of a chunk is U = (I + tril(diag(beta) M))^-1 diag(beta) (V - decay K S)."""
    t, group = v.dtype, v.shape[2] // q.shape[2]
    b, l, h, dv = v.shape
    dk, n = q.shape[3], -(-l // CHUNK)
    pad = lambda x: torch.cat([x, x.new_zeros(b, n * CHUNK - l, *x.shape[2:])], 1)  # noqa: E731
    cut = lambda x: pad(x).unflatten(1, (n, CHUNK)).movedim(3, 1)  # noqa: E731  (b, h, n, C, ...)
    q, k = (cut(x.float().repeat_interleave(group, 2)) for x in (q, k))
    v, beta = cut(v.float()), cut(beta.float())
    cum = cut(log_decay.double().clamp(min=FLOOR)).cumsum(-1)
    at = torch.arange(CHUNK, device=v.device)
    lower = at[:, None] >= at[None, :]
    decay = torch.where(lower, torch.exp(torch.where(lower, cum[..., :, None] - cum[..., None, :], 0.0)), 0.0).float()
    enter, leave, total = cum.exp().float()[..., None], (cum[..., -1:] - cum).exp().float()[..., None], cum[..., -1].exp().float()[..., None, None]
    # the inverse of a unit lower triangle: (I - A)(I + A^2)(I + A^4)..., A strictly lower
    a = torch.where(lower & (at[:, None] > at[None, :]), (k @ k.mT) * decay * beta[..., None], 0.0).double()
    eye = torch.eye(CHUNK, device=v.device, dtype=torch.float64)
    inverse, power = eye - a, a @ a
    for _ in range(5):
        inverse, power = inverse @ (eye + power), power @ power
    inverse = inverse.float() * beta[..., None, :]
    inside = (q @ k.mT) * decay * scale
    qe, ke, kl = q * enter * scale, k * enter, k * leave
    s = torch.zeros(b, h, dv, dk, device=v.device) if state is None else state
    out = []
    for i in range(n):
        u = inverse[:, :, i] @ (v[:, :, i] - ke[:, :, i] @ s.mT)
        out.append(qe[:, :, i] @ s.mT + inside[:, :, i] @ u)
        s = total[:, :, i] * s + u.mT @ kl[:, :, i]
    return torch.stack(out, 2).movedim(1, 3).flatten(1, 2)[:, :l].to(t), s


def _plain_step(s):
    """Token by token, as it is defined; the state is updated in place, as a server's cache is."""
    group, state, out = s["v"].shape[2] // s["q"].shape[2], s["state"], []
    q, k = (s[n].float().repeat_interleave(group, 2) for n in ("q", "k"))
    v, a, beta = s["v"].float(), s["log_decay"].float().exp(), s["beta"].float()
    for i in range(v.shape[1]):
        state *= a[:, i, :, None, None]
        u = beta[:, i, :, None] * (v[:, i] - (state * k[:, i, :, None, :]).sum(-1))
        state += u[..., None] * k[:, i, :, None, :]
        out.append((state * q[:, i, :, None, :]).sum(-1) * s["scale"])
    return torch.stack(out, 1).to(s["v"].dtype), state


def _codes(x, dims):
    """Codes of -127..127 and the step of each block: `dims` are a block's."""
    most = x.abs().amax(dims, keepdim=True)
    return torch.where(most > 0, torch.round(x * 127.0 / most), 0.0), most / 127.0


def _plain_round8(x):
    """Blocks of 64 consecutive values."""
    flat = x.detach().float().flatten()
    n = flat.numel()
    blocks = torch.cat([flat, flat.new_zeros(-n % 64)]).view(-1, 64)
    c, step = _codes(blocks, (1,))
    return (c * step).flatten()[:n].view(x.shape).to(x.dtype), step.flatten()


class _Rounded(torch.autograd.Function):
    """x in the forward pass; its gradient passes unchanged to x when the rounded value is used in its place."""

    @staticmethod
    def forward(ctx, x):
        return _plain_round8(x)[0]

    @staticmethod
    def backward(ctx, g):
        return g


def _plain_train(s, eight):
    leaves = [s[n] for n in LEAVES] + ([s["state"]] if "grad_state" in s else [])
    q, k, v, g, beta = leaves[:5]
    state = s.get("state")
    if eight:
        with torch.no_grad():
            o, last = _plain_delta(q, k, v, g, beta, state, s["scale"])
        o8, last8 = _plain_delta(_Rounded.apply(q), _Rounded.apply(k), _Rounded.apply(v), g, beta, state, s["scale"])
    else:
        o8, last8 = o, last = _plain_delta(q, k, v, g, beta, state, s["scale"])
    if state is None:
        return (o, *torch.autograd.grad(o8, leaves, s["grad"]))
    return (o, last, *torch.autograd.grad((o8, last8), leaves, (s["grad"], s["grad_state"])))


def _plain_scan(g, x):
    """y[t] = g[t] y[t-1] + x[t] along dim 1, by doubling."""
    l, d = g.shape[1], 1
    g = torch.cat([torch.zeros_like(g[:, :1]), g[:, 1:]], 1)
    while d < l:
        x = torch.cat([x[:, :d], g[:, d:] * x[:, :-d] + x[:, d:]], 1)
        g = torch.cat([g[:, :d], g[:, d:] * g[:, :-d]], 1)
        d *= 2
    return x


def _plain_scan8(s):
    g, x, go = s["gates"].detach().float(), s["tokens"].detach().float(), s["grad"].float()
    t = s["tokens"].dtype
    b, l, d = x.shape
    y = _plain_scan(g, x).to(t)
    # blocks of 8 timesteps x 8 channels (16 bytes)
    padded = torch.cat([y.float(), torch.zeros(b, -l % 8, d, device=y.device)], 1).view(b, -1, 8, d // 8, 8)
    c, step = _codes(padded, (2, 4))
    y8 = (c * step).view(b, -1, d)[:, :l]
    nothing = torch.zeros_like(g[:, :1])
    dx = _plain_scan(torch.cat([g[:, 1:], nothing], 1).flip(1), go.flip(1)).flip(1)
    dg = dx * torch.cat([nothing, y8[:, :-1]], 1)
    return y, dg.to(t), dx.to(t)


def run(state):
    s, op = state, state["op"]
    if own:
        import fpscan_b200 as fp
        if op == "step":
            return fp.gated_delta_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], scale=s["scale"]), s["state"]
        if op == "prefill":
            return fp.gated_delta_forward(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], initial_state=s.get("state"),
                                          scale=s["scale"], return_state=True)
        if op == "round8":
            codes, steps = fp.quantize8(s["x"])
            return fp.dequantize8(codes, steps, s["x"].dtype), steps
        if op == "scan8":
            y = fp.pscan_channels_last(s["gates"], s["tokens"], checkpoint8=True)
            return (y, *torch.autograd.grad(y, (s["gates"], s["tokens"]), s["grad"]))
        leaves = [s[n] for n in LEAVES]
        if "grad_state" not in s:
            o = fp.gated_delta(*leaves, scale=s["scale"], checkpoint8=op == "train8")
            return (o, *torch.autograd.grad(o, leaves, s["grad"]))
        o, last = fp.gated_delta(*leaves, initial_state=s["state"], scale=s["scale"], return_state=True, checkpoint8=op == "train8")
        return (o, last, *torch.autograd.grad((o, last), leaves + [s["state"]], (s["grad"], s["grad_state"])))
    if op == "step":
        return _plain_step(s)
    if op == "prefill":
        return _plain_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s.get("state"), s["scale"])
    if op == "round8":
        return _plain_round8(s["x"])
    if op == "scan8":
        return _plain_scan8(s)
    return _plain_train(s, op == "train8")


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "fp32" else 2
    if op == "round8":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (e + 1 + 1 + e) + n // 64 * 8, "flops": n * 5}  # x, the codes twice, the values
    if op == "scan8":
        n = case["batch"] * case["seqlen"] * case["dim"]
        return {"bytes": n * (8 * e - e + 2) + n // 64 * 8, "flops": n * 10}  # 2 in, 1 out; 2 in, 2 out; the codes twice
    b, l, hk, dk, dv = (case[n] for n in ("batch", "seqlen", "key_heads", "dk", "dv"))
    h = hk * case["group"]
    ins = b * l * (2 * hk * dk + h * dv + 2 * h) * e
    out = b * l * h * dv * e
    state = b * h * dk * dv * 4
    unit = b * l * h * dk * dv  # one product of a token with the state
    if op == "step":
        return {"bytes": ins + out + 2 * state, "flops": 7 * unit}
    if op == "prefill":
        return {"bytes": ins + out + 2 * state, "flops": 7 * unit}
    # forward: inputs, output; backward: inputs (in 8 bits: written and read), output's gradient, inputs' gradients
    again = ins if op == "train" else b * l * (2 * hk * dk + h * dv) * 2
    return {"bytes": 2 * ins + again + 2 * out + (4 * state if case["state"] else 0), "flops": 24 * unit}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_tokens(q, k, v, a, beta, state, scale):
    """Token by token: the definition. All (b, l, h, ...) in 64 bits."""
    out = []
    for q, k, v, a, beta in zip(*(x.unbind(1) for x in (q, k, v, a, beta))):
        held = a[..., None, None] * state
        u = beta[..., None] * (v - torch.einsum("bhvk,bhk->bhv", held, k))
        state = held + u[..., :, None] * k[..., None, :]
        out.append(scale * torch.einsum("bhvk,bhk->bhv", state, q))
    return torch.stack(out, 1), state


def _exact_round(x):
    """Nearest multiples, ties to even, of a block's largest magnitude over 127."""
    flat = x.detach().double().reshape(-1)
    n = flat.numel()
    rows = torch.nn.functional.pad(flat, (0, -n % 64)).reshape(-1, 64)
    step = rows.abs().max(1, keepdim=True).values / 127
    return (torch.round(rows / step.clamp(min=1e-300)) * step).reshape(-1)[:n].reshape(x.shape), step.reshape(-1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "round8":
        x = s["x"]
        if x.dtype == torch.float32:
            return None  # a tie's side goes by the rounding of the quotient: the codes are defined in 32 bits
        return _exact_round(x)
    if op == "scan8":
        g, x, go = (s[n].detach().double() for n in ("gates", "tokens", "grad"))
        b, l, d = x.shape
        y, dx, h = torch.empty_like(x), torch.empty_like(x), torch.zeros_like(x[:, 0])
        for i in range(l):
            h = g[:, i] * h + x[:, i]
            y[:, i] = h
        h = torch.zeros_like(h)
        for i in range(l - 1, -1, -1):
            h = go[:, i] + (g[:, i + 1] * h if i + 1 < l else 0)
            dx[:, i] = h
        dg = torch.zeros_like(x)
        held = y.to(s["tokens"].dtype).double()  # what is kept is the output, as it is returned
        for t in range(0, l, 8):
            tile = held[:, t:t + 8].unflatten(2, (-1, 8))
            step = tile.abs().amax((1, 3), keepdim=True) / 127
            held[:, t:t + 8] = (torch.round(tile / step.clamp(min=1e-300)) * step).flatten(2)
        dg[:, 1:] = dx[:, 1:] * held[:, :-1]
        return y, dg, dx
    group, scale = case["group"], s["scale"]
    b, l, h, dv = s["v"].shape
    if l > 20000:
        return None
    wide = [x.detach().double() for x in (s[n] for n in LEAVES)]
    state = s["state"].detach().double() if "state" in s else torch.zeros(b, h, dv, case["dk"], device="cuda", dtype=torch.float64)

    def piece(x, i, state):
        q, k, v, g, beta = (t[:, i:i + 64] for t in x)
        return _exact_tokens(q.repeat_interleave(group, 2), k.repeat_interleave(group, 2), v, g.exp(), beta, state, scale)

    out, starts = [], []
    for i in range(0, l, 64):
        o, state = piece(wide, i, state)
        out.append(o)
    o = torch.cat(out, 1)
    if op in ("step", "prefill"):
        return o, state
    last, used = state, wide
    if op == "train8":  # the backward pass sees q, k and v as the checkpoints give them back, in their type
        used = [_exact_round(x)[0].to(x.dtype).double() for x in (s["q"], s["k"], s["v"])] + wide[3:]
    state = s["state"].detach().double() if "state" in s else torch.zeros_like(last)
    for i in range(0, l, 64):
        starts.append(state)
        state = piece(used, i, state)[1]
    d_state = s["grad_state"].double() if "grad_state" in s else torch.zeros_like(last)
    grads, go = [], s["grad"].double()
    for i in range(0, l, 64)[::-1]:
        with torch.enable_grad():
            x = [t[:, i:i + 64].clone().requires_grad_() for t in used]
            s0 = starts[i // 64].clone().requires_grad_()
            o1, s1 = piece(x, 0, s0)
            *d, d_state = torch.autograd.grad((o1, s1), x + [s0], (go[:, i:i + 64], d_state))
        grads.append(d)
    grads = [torch.cat(x[::-1], 1) for x in zip(*grads)]
    return (o, last, *grads, d_state) if "grad_state" in s else (o, *grads)
