"""What the second set of sequence operators is timed on: linear attention with a decay for each head, the gated projection
of a feed-forward block, and AdamW over all of a readout's variables at once.

Every case is a plain dict.  ``op`` names the operator, ``call`` how it is used: ``fwd`` (evaluation), ``train`` (the output
and every gradient), ``tick`` (one time step, the state updated in place) or ``step`` (one update of the optimizer);
``dtype`` is that of the activations or variables.  Sequences are time-major, [ticks ``T``, batch ``B``, heads, channels], as
the column's rollouts are.  The sizes are those of the package's configurations (66,000 neurons, 500 ticks, batches 1, 5 and
32), an odd-sized network's (12,007 neurons, 120 ticks, batch 3), the readout example's, and a readout's own widths.

Plain forms are elementary torch operations in 32 bits, rounded once to the type of the output.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64                 # ticks that the plain attention takes together
BLOCK = 256                # values that share a scale where moments are held in 8 bits
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.99, 1e-8, 0.01


def listed():
    return [
        # one tick of batch 32 beside the column: the state is read and written once
        dict(name="attention_tick", op="attention", call="tick", T=1, B=32, H=8, G=8, K=64, V=64, dtype="bf16", ragged=False),
        # one long recording, 8 s
        dict(name="attention_prompt", op="attention", call="fwd", T=8000, B=1, H=16, G=16, K=128, V=128, dtype="bf16", ragged=False),
        # an odd-sized network's training window in full precision, keys and values shared by heads
        dict(name="attention_shared", op="attention", call="train", T=120, B=3, H=6, G=2, K=24, V=40, dtype="f32", ragged=True),
        # a training window of batch 32, trials of their own lengths
        dict(name="attention_train", op="attention", call="train", T=500, B=32, H=8, G=8, K=128, V=128, dtype="bf16", ragged=True),
        # one tick of batch 5 through a block: the weights are read for few rows
        dict(name="gated_tick", op="gated", call="fwd", M=5, K=1024, N=4096, act="silu", bias=False, dtype="bf16"),
        # an odd-sized block over a short window in full precision
        dict(name="gated_ragged", op="gated", call="train", M=360, K=257, N=683, act="gelu", bias=True, dtype="f32"),
        # evaluation of a training window, batch 5
        dict(name="gated_window", op="gated", call="fwd", M=2500, K=512, N=1365, act="silu", bias=True, dtype="f16"),
        # a training window of batch 32: the largest
        dict(name="gated_train", op="gated", call="train", M=16000, K=1024, N=4096, act="silu", bias=False, dtype="bf16"),
        # the readout example's variables: latency
        dict(name="adamw_example", op="adamw", call="step", neurons=400, width=64, channels=128, outputs=4, bits=32, dtype="f32"),
        # a readout of the whole column
        dict(name="adamw_column", op="adamw", call="step", neurons=66000, width=512, channels=1024, outputs=10, bits=32, dtype="f32"),
        # its moments in 8 bits
        dict(name="adamw_column8", op="adamw", call="step", neurons=66000, width=512, channels=1024, outputs=10, bits=8, dtype="f32"),
        # an odd-sized network's readout with variables in 16 bits
        dict(name="adamw_odd", op="adamw", call="step", neurons=12007, width=256, channels=512, outputs=7, bits=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "gated", "adamw"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32", "f16"]))
    if op == "gated":
        K, N = _log(rng, 32, 4096), _log(rng, 16, 8192)
        M = _log(rng, 1, max(1, min(16000, 40_000_000_000 // (K * N))))
        return dict(c, call=rng.choice(["fwd", "train"]), M=M, K=K, N=N, act=rng.choice(["silu", "gelu", "relu"]), bias=rng.random() < 0.5)
    if op == "adamw":
        return dict(c, call="step", neurons=_log(rng, 100, 66000), width=_log(rng, 32, 512), channels=_log(rng, 64, 1024),
                    outputs=rng.randint(2, 40), bits=rng.choice([8, 32]))
    call = rng.choice(["fwd", "train", "train", "tick"])
    B, G = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 8])
    H = G * rng.choice([1, 1, 2, 4])
    K, V = rng.choice([16, 32, 64, 64, 128, rng.randint(8, 128)]), rng.choice([16, 32, 64, 64, 128, rng.randint(8, 128)])
    T = 1 if call == "tick" else _log(rng, 2, max(2, min(8000, 1_000_000_000 // (B * H * K * V))))
    return dict(c, call=call, T=T, B=B, H=H, G=G, K=K, V=V, ragged=call != "tick" and rng.random() < 0.5)


def _shapes(c):
    """The variables of a readout (16 states, 4 taps, steps of rank 16)."""
    n, w, ch, o = c["neurons"], c["width"], c["channels"], c["outputs"]
    return [(n,), (n,), (w, n), (w,), (w,), (w,), (2 * ch, w), (ch, 4), (ch,), (48, ch), (ch, 16), (ch,), (ch, 16), (ch,),
            (w, ch), (w,), (w,), (w,), (o, w), (o,)]


# -------------------------------------------------------------------- the inputs ----
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, f32 = TYPES[c["dtype"]], torch.float32
    train = c["call"] == "train"

    def randn(*shape, scale=1.0, dtype=dt, wrt=True):
        t = (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)
        return t.requires_grad_(True) if train and wrt else t

    s = dict(case=c)
    if c["op"] == "attention":
        T, B, H, G, K, V = (c[k] for k in "TBHGKV")
        lead = (B,) if c["call"] == "tick" else (T, B)
        s["q"], s["k"], s["v"] = randn(*lead, H, K), randn(*lead, G, K), randn(*lead, G, V)
        # heads that remember from four ticks to four thousand
        s["decay"] = -torch.exp(torch.linspace(math.log(0.25), math.log(0.00025), H, device=DEV))
        s["state"] = randn(B, H, K, V, dtype=f32)
        s["len"] = None
        if c["ragged"]:
            s["len"] = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
            s["len"][0] = T
        if train:
            s["dy"], s["dstate"] = randn(T, B, H, V, wrt=False), randn(B, H, K, V, dtype=f32, wrt=False)
    elif c["op"] == "gated":
        M, K, N = c["M"], c["K"], c["N"]
        s["x"], s["w"] = randn(M, K), randn(2 * N, K, scale=K ** -0.5)
        s["b"] = randn(2 * N, scale=0.1) if c["bias"] else None
        if train:
            s["dy"] = randn(M, N, wrt=False)
    else:
        shapes = _shapes(c)
        s["p"] = [randn(*shape, scale=0.1) for shape in shapes]
        # gradients of many sizes, and moments as hundreds of steps leave them
        size = [1e-3 * torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV)) for shape in shapes]
        s["g"] = [(torch.randn(z.shape, generator=g, device=DEV) * z).to(dt) for z in size]
        s["done"] = 300 + int(seed) % 100
        s["noise"] = 1_000_003 * int(seed) + 29
        s["m"] = [0.3 * torch.randn(z.shape, generator=g, device=DEV) * z for z in size]
        s["v"] = [z * z * (0.5 + torch.rand(z.shape, generator=g, device=DEV)) for z in size]
        if c["bits"] == 8:
            for name, top, code in (("m", 127, torch.int8), ("v", 255, torch.uint8)):
                s[name] = [_held(x, top, code, g) for x in s[name]]
        if own:   # the optimizer that a program keeps
            from v1_glif_model_amd.optim import AdamW
            s["opt"] = AdamW(s["p"], LR, BETA1, BETA2, EPS, DECAY, state_bits=c["bits"], seed=s["noise"])
            s["opt"].load_state_dict(dict(iterations=s["done"], first=s["m"], second=s["v"]))
    return s


# ---------------------------------------------------------------------- one pass ----
def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    c = s["case"]
    if c["op"] == "adamw":
        s["opt"].apply_gradients(s["g"])
        return (s["p"], *s["opt"].moments())
    from v1_glif_model_amd import sequence as seq
    if c["op"] == "gated":
        y = seq.gated_linear(s["x"], s["w"], s["b"], activation=c["act"])
        return y if c["call"] == "fwd" else _grads(y, (s["x"], s["w"], s["b"]), s["dy"])
    if c["call"] == "tick":
        return seq.linear_attention_step(s["q"], s["k"], s["v"], s["state"], s["decay"]), s["state"]
    out = seq.linear_attention(s["q"], s["k"], s["v"], s["decay"], initial_state=s["state"], lengths=s["len"])
    return out if c["call"] == "fwd" else _grads(out, (s["q"], s["k"], s["v"], s["state"]), (s["dy"], s["dstate"]))


def _grads(out, wrt, dout):
    out, dout = (out, dout) if isinstance(out, tuple) else ((out,), (dout,))
    return (*(o.detach() for o in out), *torch.autograd.grad(out, [t for t in wrt if t is not None], dout))


@torch.no_grad()
def _plain(s):
    return {"attention": _plain_attention, "gated": _plain_gated, "adamw": _plain_adamw}[s["case"]["op"]](s)


def _powers(decay, n):
    """exp(decay * n) for whole n >= 0 (0 elsewhere), in 64 bits up to the rounding of the result: decay [H], n [...] gives
    [H, ...]."""
    p = torch.exp(decay.double().reshape(-1, *[1] * n.dim()) * n.clamp(min=0).double())
    return torch.where(n >= 0, p, torch.zeros_like(p)).float()


def _causal(q, k, v, decay):
    """sum over j <= i of exp(decay (i - j)) (q_i . k_j) v_j: q, k [B, H, T, K], v [B, H, T, V], in chunks of ticks whose
    states are joined by one product over the chunks."""
    B, H, T, K = q.shape
    n = (T + CHUNK - 1) // CHUNK
    cut = lambda t: torch.nn.functional.pad(t, (0, 0, 0, n * CHUNK - T)).reshape(B, H, n, CHUNK, -1)  # noqa: E731
    q, k, v = cut(q), cut(k), cut(v)
    i, c = torch.arange(CHUNK, device=DEV), torch.arange(n, device=DEV)
    inside = (q @ k.transpose(-1, -2).contiguous()) * _powers(decay, i[:, None] - i)[:, None] @ v
    ends = (k * _powers(decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    starts = _powers(decay, (c[:, None] - c - 1) * CHUNK) @ ends.reshape(B, H, n, -1)       # the state before each chunk
    across = (q * _powers(decay, i + 1)[:, None, :, None]) @ starts.reshape(ends.shape)
    return (inside + across).reshape(B, H, n * CHUNK, -1)[:, :, :T]


def _plain_attention(s):
    c, decay = s["case"], s["decay"]
    dt, K, H, G = s["q"].dtype, c["K"], c["H"], c["G"]
    scale = K ** -0.5
    q, k, v, h0 = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    if c["call"] == "tick":
        k, v = (t.repeat_interleave(H // G, 1) for t in (k, v))
        h0.copy_(_powers(decay, torch.ones((), device=DEV))[:, None, None] * h0 + k[..., None] * v[..., None, :])
        return (scale * (q[..., None] * h0).sum(-2)).to(dt), h0
    T = q.shape[0]
    heads = lambda t: t.permute(1, 2, 0, 3).repeat_interleave(H // t.shape[2], 1)  # noqa: E731  [B, H, T, channels]
    q, k, v = heads(q) * scale, heads(k), heads(v)
    t = torch.arange(T, device=DEV)
    end = s["len"].long() if s["len"] is not None else torch.full((c["B"],), T, device=DEV)
    live = (t < end[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, torch.zeros((), device=DEV)) for x in (q, k, v))
    after = _powers(decay, t + 1)[:, :, None]                                               # [H, T, 1]
    left = _powers(decay, end[:, None] - 1 - t).transpose(0, 1)[..., None]                  # [B, H, T, 1]
    whole = _powers(decay, end).t()[..., None, None]                                        # [B, H, 1, 1]
    y = _causal(q, k, v, decay) + (q * after) @ h0
    last = whole * h0 + (k * left).transpose(-1, -2).contiguous() @ v
    back = lambda x: x.permute(2, 0, 1, 3).to(dt).contiguous()  # noqa: E731
    if c["call"] == "fwd":
        return back(y), last
    dy, dlast = torch.where(live, heads(s["dy"].float()), torch.zeros((), device=DEV)), s["dstate"]
    turn = lambda *xs: [x.flip(2) for x in xs]  # noqa: E731  time backwards
    dq = _causal(dy, v, k, decay) + (dy * after) @ h0.transpose(-1, -2).contiguous()
    dk = _causal(*turn(v, dy, q), decay).flip(2) + (v * left) @ dlast.transpose(-1, -2).contiguous()
    dv = _causal(*turn(k, q, dy), decay).flip(2) + (k * left) @ dlast
    dq, dk, dv = (torch.where(live, x, torch.zeros((), device=DEV)) for x in (scale * dq, dk, dv))
    dk, dv = (x.unflatten(1, (G, H // G)).sum(2) for x in (dk, dv))
    dh0 = whole * dlast + (q * after).transpose(-1, -2).contiguous() @ dy
    return back(y), last, back(dq), back(dk), back(dv), dh0


def _plain_act(p, act):
    """The activation and its slope."""
    if act == "relu":
        return torch.relu(p), (p > 0).float()
    if act == "gelu":
        half = 0.5 * (1.0 + torch.erf(p * 0.5 ** 0.5))
        return p * half, half + p * torch.exp(-0.5 * p * p) * (2.0 * math.pi) ** -0.5
    q = torch.sigmoid(p)
    return p * q, q * (1.0 + p * (1.0 - q))


def _plain_gated(s):
    c, x, w = s["case"], s["x"].float(), s["w"].float()
    dt, pre = s["x"].dtype, x @ w.t()
    if s["b"] is not None:
        pre = pre + s["b"].float()
    gate, up = pre.split(c["N"], -1)
    on, slope = _plain_act(gate, c["act"])
    y = (on * up).to(dt)
    if c["call"] == "fwd":
        return y
    dy = s["dy"].float()
    dp = torch.cat([dy * up * slope, dy * on], -1)
    grads = [(dp @ w).to(dt), (dp.t() @ x).to(dt)] + ([dp.sum(0).to(dt)] if s["b"] is not None else [])
    return (y, *grads)


def _philox(seed, first, n):
    """Words first .. first + n - 1 of the Philox4x32-10 stream of ``seed``, as int64: word i is word i % 4 of the block of
    counter i // 4.  ``first`` is a multiple of 4."""
    low = 0xFFFFFFFF
    blk = torch.arange(first // 4, (first + n + 3) // 4, device=DEV)
    c = [blk & low, blk >> 32, torch.zeros_like(blk), torch.zeros_like(blk)]
    k0, k1 = seed & low, (seed >> 32) & low
    for r in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # modulo 2^64: the bits are those of the product
        c = [(b >> 32) & low ^ c[1] ^ k0, b & low, (a >> 32) & low ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, -1).reshape(-1)[:n]


def _level(code, top):
    """What a code stands for beside its block's scale: squares of 127ths for first moments, fourth powers of 255ths for
    second ones."""
    r = code * torch.tensor(1.0 / top, dtype=torch.float32, device=DEV)
    return r * r.abs() if top == 127 else (r * r) * (r * r)


def _decode(held, top):
    code, scale = held
    return _level(code.float(), top) * scale.repeat_interleave(BLOCK)[:code.numel()].reshape(code.shape)


def _encode(x, held, top, u):
    """x into codes and scales: to the code below or above by the 16-bit random number u, so that the mean is kept; what is
    not 0 of a second moment does not become 0."""
    code, scale = held
    n = x.numel()
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).reshape(-1, BLOCK)
    most = flat.abs().amax(1)
    fine = torch.isfinite(most) & (most >= torch.finfo(torch.float32).tiny)
    part = flat.abs() * (1.0 / most)[:, None]
    root = torch.sqrt(part) if top == 127 else torch.sqrt(torch.sqrt(part))
    below = torch.floor(root * top).clamp(max=top - 1)
    a, b = _level(below, top), _level(below + 1.0, top)
    up = u.reshape(-1, BLOCK).float() * (b - a) < (part - a) * 65536.0
    new = below + up
    if top == 255:
        new = torch.where(flat > 0, new.clamp(min=1.0), new)
    new = torch.where(fine[:, None], new, torch.zeros_like(new)) * (torch.sign(flat) if top == 127 else 1.0)
    code.copy_(new.reshape(-1)[:n].reshape(code.shape).to(code.dtype))
    scale.copy_(most)


def _held(x, top, code, g):
    """x as codes and scales."""
    n = (x.numel() + BLOCK - 1) // BLOCK
    held = torch.empty(x.shape, dtype=code, device=DEV), torch.empty(n, device=DEV)
    _encode(x, held, top, torch.randint(0, 65536, (n * BLOCK,), generator=g, device=DEV))
    return held


def _plain_adamw(s):
    c = s["case"]
    s["done"] += 1
    t, eight = s["done"], c["bits"] == 8
    step, root = LR / (1.0 - BETA1 ** t), math.sqrt(1.0 - BETA2 ** t)
    at = [(p.numel() + BLOCK - 1) // BLOCK * BLOCK for p in s["p"]]
    first = (t - 1) * sum(at)
    ms, vs = [], []
    for i, (p, g) in enumerate(zip(s["p"], s["g"])):
        g = g.float()
        m, v = (_decode(s["m"][i], 127), _decode(s["v"][i], 255)) if eight else (s["m"][i], s["v"][i])
        m = m * BETA1 + g * (1.0 - BETA1)
        v = v * BETA2 + (g * g) * (1.0 - BETA2)
        p.copy_((p.float() * (1.0 - LR * DECAY) - step * (m / (torch.sqrt(v) / root + EPS))).to(p.dtype))
        if eight:
            word = _philox(s["noise"], first, at[i])
            first += at[i]
            _encode(m, s["m"][i], 127, word & 0xFFFF)
            _encode(v, s["v"][i], 255, word >> 16)
            m, v = _decode(s["m"][i], 127), _decode(s["v"][i], 255)
        else:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
        ms.append(m)
        vs.append(v)
    return s["p"], ms, vs


# -------------------------------------------------------------- the work of a pass ----
def work(case):
    c = case
    size, train = TYPES[c["dtype"]].itemsize, c["call"] == "train"
    if c["op"] == "adamw":
        n = sum(math.prod(shape) for shape in _shapes(c))
        # variables and gradients, and the moments: in 8 bits those are read and written and given back as values
        state = 16 if c["bits"] == 32 else 4 + 16 / BLOCK + 8
        return dict(bytes=n * (3 * size + state), flops=n * 14)
    if c["op"] == "gated":
        M, K, N = c["M"], c["K"], c["N"]
        b = M * K + 2 * N * K + M * N + (2 * N if c["bias"] else 0)
        return dict(bytes=(2 * b if train else b) * size, flops=4 * M * K * N * (3 if train else 1))
    T, B, H, G, K, V = (c[k] for k in "TBHGKV")
    ticks = T + (B - 1) * T / 2 if c["ragged"] else T * B      # trials of any length, half of the window on average
    rows = ticks * (H * (K + V) + G * (K + V)) * size
    state = 2 * B * H * K * V * 4
    return dict(bytes=2 * (rows + state) if train else rows + state, flops=ticks * H * K * V * (14 if train else 4))


# ----------------------------------------------------------- the definitions in 64 bits ----
def exact(case, seed):
    """What ``run`` gives for these inputs, in 64 bits and one tick at a time."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "gated": _exact_gated, "adamw": _exact_adamw}[case["op"]](case, s)


def _exact_attention(c, s):
    q, k, v, h = (s[n].detach().double() for n in ("q", "k", "v", "state"))
    lam, scale, each = torch.exp(s["decay"].double())[:, None, None], c["K"] ** -0.5, c["H"] // c["G"]
    if c["call"] == "tick":
        k, v = k.repeat_interleave(each, 1), v.repeat_interleave(each, 1)
        h = lam * h + k.unsqueeze(-1) * v.unsqueeze(-2)
        return scale * (q.unsqueeze(-2) @ h).squeeze(-2), h
    k, v = k.repeat_interleave(each, 2), v.repeat_interleave(each, 2)
    T, train = c["T"], c["call"] == "train"
    ends = [T] * c["B"] if s["len"] is None else s["len"].tolist()
    on = torch.tensor([[t < e for e in ends] for t in range(T)], device=DEV)[..., None, None, None]
    y, dq = torch.zeros(*q.shape[:-1], c["V"], dtype=torch.float64, device=DEV), torch.zeros_like(q)
    dy = s["dy"].double() if train else None
    for t in range(T):
        h = torch.where(on[t], lam * h + k[t].unsqueeze(-1) * v[t].unsqueeze(-2), h)
        y[t] = scale * ((q[t].unsqueeze(-2) @ h).squeeze(-2) * on[t][..., 0])
        if train:
            dq[t] = scale * ((h @ dy[t].unsqueeze(-1)).squeeze(-1) * on[t][..., 0])
    if not train:
        return y, h
    dk, dv, dh = torch.zeros_like(k), torch.zeros_like(v), s["dstate"].double()
    for t in reversed(range(T)):
        inner = dh + scale * q[t].unsqueeze(-1) * dy[t].unsqueeze(-2)
        dk[t] = (inner @ v[t].unsqueeze(-1)).squeeze(-1) * on[t][..., 0]
        dv[t] = (k[t].unsqueeze(-2) @ inner).squeeze(-2) * on[t][..., 0]
        dh = torch.where(on[t], lam * inner, dh)
    dk, dv = dk.unflatten(2, (c["G"], each)).sum(3), dv.unflatten(2, (c["G"], each)).sum(3)
    return y, h, dq, dk, dv, dh


def _exact_gated(c, s):
    x, w, N = s["x"].detach().double(), s["w"].detach().double(), c["N"]
    g, u = x @ w[:N].t(), x @ w[N:].t()
    if s["b"] is not None:
        g, u = g + s["b"][:N].detach().double(), u + s["b"][N:].detach().double()
    if c["act"] == "relu":
        a, da = g.clamp(min=0.0), (g > 0).double()
    elif c["act"] == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        a, da = g * cdf, cdf + g * torch.exp(-g * g / 2.0) / math.sqrt(2.0 * math.pi)
    else:
        cdf = 1.0 / (1.0 + torch.exp(-g))
        a, da = g * cdf, cdf + g * cdf * (1.0 - cdf)
    if c["call"] == "fwd":
        return a * u
    dy = s["dy"].double()
    dg, du = dy * u * da, dy * a
    out = [a * u, dg @ w[:N] + du @ w[N:], torch.cat([dg.t() @ x, du.t() @ x])]
    return (*out, torch.cat([dg.sum(0), du.sum(0)])) if s["b"] is not None else tuple(out)


def _exact_adamw(c, s):
    t, ps, ms, vs = s["done"] + 1, [], [], []
    for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        p, g = p.double(), g.double()
        if c["bits"] == 8:
            (cm, sm), (cv, sv) = m, v
            spread = lambda z: z.double().repeat_interleave(BLOCK)[:p.numel()].reshape(p.shape)  # noqa: E731
            cm, cv = cm.double() / 127.0, cv.double() / 255.0
            m, v = cm * cm.abs() * spread(sm), cv ** 4 * spread(sv)
        m = BETA1 * m.double() + (1.0 - BETA1) * g
        v = BETA2 * v.double() + (1.0 - BETA2) * g * g
        hat = (v / (1.0 - BETA2 ** t)).sqrt()
        ps.append(p - LR * DECAY * p - LR * (m / (1.0 - BETA1 ** t)) / (hat + EPS))
        ms.append(m)
        vs.append(v)
    # moments that are rounded to 8 bits by random numbers have no values in 64 bits
    return (ps, ms, vs) if c["bits"] == 32 else (ps, None, None)
