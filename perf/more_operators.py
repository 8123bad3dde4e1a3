"""More operators on caller tensors (redukt_amd.ops): what they are measured on.

The parts of a selective state-space layer in 8 bits, each with its plain form in elementary
torch operations (`own` false) and as a user calls the framework's kernel (`own` true):

  scan_chunk  the gated linear recurrence over whole packed sequences.  With
              s = softplus(dt + bias), a channel's state h [n] takes a token as
                  h <- e^(s A) h + s x B,    y = C.h + D x,    out = y silu(z)
  scan_step   the same for one token of each of n streams, states in a pool of slots
  scan_grad   its backward pass: the gradients of everything that goes in
  quantize    e4m3 codes with one f32 scale for each 128 columns of a row, or of 128 rows
  matmul      the product of such codes
  sample      the next token: temperature, top-k, top-p, min-p, given random numbers

`listed()` holds cases of each from one token to the largest; `draw()` gives more of the same
ranges.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
ONE = 2.0 ** 42      # the weight of the largest logit: weights are whole numbers, so their sums are exact


def listed():
    def scan(name, op, seqs, tokens, channels, n, groups, dtype, initial, gate):
        return {"name": name, "op": op, "seqs": seqs, "tokens": tokens, "channels": channels, "n": n, "groups": groups,
                "dtype": dtype, "initial": initial, "gate": gate}

    def quantize(name, rows, cols, block_rows, dtype):
        return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "block_rows": block_rows, "dtype": dtype}

    def matmul(name, m, n, k, dtype, bias):
        return {"name": name, "op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}

    def sample(name, rows, vocab, dtype, filters):
        return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters}

    return [
        # a short prompt of one stream in 32 bits, the layer of Mamba-130M
        scan("scan_200_f32", "scan_chunk", 1, 200, 1536, 16, 1, "f32", False, True),
        # a batch of prompts of very different lengths, continued from earlier states
        scan("scan_37_ragged", "scan_chunk", 37, 20011, 1536, 16, 1, "bf16", True, True),
        # one interactive stream: latency only
        scan("step_1", "scan_step", 1, 1, 1536, 16, 1, "bf16", True, True),
        # a large lockstep batch: the states' bytes
        scan("step_1000_f16", "scan_step", 1000, 1000, 1536, 16, 1, "f16", True, True),
        # a training step's layer on four short segments, in 32 bits
        scan("grad_4_f32", "scan_grad", 4, 1030, 768, 16, 1, "f32", True, True),
        # a training step's layer on one long document, two groups of B and C
        scan("grad_8192", "scan_grad", 1, 8192, 1536, 16, 2, "bf16", False, True),
        # the activations of one token
        quantize("quantize_1", 1, 768, 1, "f32"),
        # the inner activations of a long prompt
        quantize("quantize_8191", 8191, 4096, 1, "bf16"),
        # the head for one stream: the weights are read once
        matmul("matmul_1", 1, 50280, 768, "f32", False),
        # a projection for a long prompt: the matrix cores' rate
        matmul("matmul_8192", 8192, 8192, 4096, "bf16", True),
        # the next token of one stream
        sample("sample_1", 1, 50280, "f32", "all"),
        # the next tokens of a large batch, each row with settings of its own
        sample("sample_1000", 1000, 50280, "bf16", "all"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["scan_chunk", "scan_chunk", "scan_step", "scan_grad", "scan_grad", "quantize", "matmul", "matmul", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("scan"):
        n = rng.choice([8, 16, 16, 16, 32, 64])
        groups = rng.choice([1, 1, 1, 2])
        channels = 64 * groups * rng.choice([1, 2, 3, 6, 8, 12]) if groups > 1 else rng.choice([192, 768, 1536, _log_int(rng, 17, 1536)])
        most = {"scan_chunk": 20011, "scan_grad": 8192, "scan_step": 1000}[op]
        most = max(1, min(most, most * 1536 * 16 // (channels * n)))
        tokens = _log_int(rng, 1, most)
        seqs = tokens if op == "scan_step" else _log_int(rng, 1, min(64, tokens))
        return {"op": op, "seqs": seqs, "tokens": tokens, "channels": channels, "n": n, "groups": groups, "dtype": dtype,
                "initial": op == "scan_step" or rng.random() < 0.5, "gate": rng.random() < 0.8}
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 8191), "cols": rng.choice([64, 200, 768, 1000, 1536, _log_int(rng, 16, 4096)]),
                "block_rows": rng.choice([1, 1, 128]), "dtype": dtype}
    if op == "matmul":
        while True:
            m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 50280), rng.choice([16 * _log_int(rng, 1, 512), 128 * _log_int(rng, 1, 64)])
            if m * n * k <= 8192 * 8192 * 4096 and m * n <= 1 << 26:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
    vocab = rng.choice([256, 1000, 50280, _log_int(rng, 2, 131072)])
    return {"op": op, "rows": _log_int(rng, 1, max(1, min(1000, 1000 * 50280 // vocab))), "vocab": vocab, "dtype": dtype,
            "filters": rng.choice(["all", "all", "none", "top_k", "top_p", "min_p"])}


# ---- inputs ----

def _lengths(case):
    """The sequences' lengths, at least one token each: most of them short, a few long."""
    seqs, left = case["seqs"], case["tokens"] - case["seqs"]
    share = (np.arange(seqs) * 7 % seqs + 1.0) ** 2
    extra = np.floor(share / share.sum() * left).astype(np.int64)
    extra[0] += left - extra.sum()
    return (extra + 1).tolist()


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scan_inputs(case, seed):
    """A layer as it is initialized (A near -1 to -n, time steps of 1/1000 to 1/10 behind the bias), activations
    as its convolution and projections give them."""
    g = _generator(seed)
    T, ch, n, dtype = case["tokens"], case["channels"], case["n"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    step = torch.exp(torch.rand(ch, generator=g, device="cuda") * 4.6 - 6.9)
    x = {"x": torch.nn.functional.silu(randn(T, ch) * 1.5).to(dtype), "dt": (0.7 * randn(T, ch)).to(dtype),
         "a": -torch.arange(1, n + 1, device="cuda") * torch.exp(0.1 * randn(ch, n)),
         "b": randn(T, case["groups"], n).to(dtype), "c": randn(T, case["groups"], n).to(dtype),
         "d": 1.0 + 0.1 * randn(ch), "dt_bias": step + torch.log(-torch.expm1(-step)),
         "z": randn(T, ch).to(dtype) if case["gate"] else None}
    if case["op"] == "scan_grad":
        x["dout"] = randn(T, ch).to(dtype)
        x["dfinal"] = 0.1 * randn(case["seqs"], ch, n) if case["initial"] else None
    return x


def _states(case, slots, seed):
    return 0.5 * torch.randn(slots, case["channels"], case["n"], generator=_generator(seed + 77), device="cuda")


def _slots(n, seed):
    """n of the n + 3 slots of a pool, in an order of their own."""
    return torch.from_numpy(np.random.default_rng(seed).permutation(n + 3)[:n].astype(np.int32)).cuda()


def _activations(case, seed):
    """Rows as a norm leaves them, of different magnitudes, a few columns much larger."""
    g = _generator(seed)
    x = torch.randn(case["rows"], case["cols"], generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(case["rows"], 1, generator=g, device="cuda"))
    x[:, ::97] *= 8.0
    return x.to(DTYPES[case["dtype"]])


def _product_inputs(case, seed):
    """Codes that use e4m3's range up to about 448, scales of activations and weights."""
    g = _generator(seed)
    m, n, k = case["m"], case["n"], case["k"]
    kb, nb = -(-k // 128), -(-n // 128)

    def codes(rows):
        return (torch.randn(rows, k, generator=g, device="cuda") * 110.0).clamp(-448, 448).to(F8)

    def scales(rows, size):
        return torch.exp(0.3 * torch.randn(rows, kb, generator=g, device="cuda")) * size

    return {"x": codes(m), "w": codes(n), "sx": scales(m, 1.0 / 110.0), "sw": scales(nb, 1.0 / (110.0 * k ** 0.5)),
            "bias": 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None}


def _logits(case, seed):
    """Logits as a head gives them: a bulk, a few hundred likely tokens, some of them masked."""
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    likely = torch.randint(0, vocab, (rows, min(vocab, 300)), generator=g, device="cuda")
    x.scatter_add_(1, likely, 6.0 * torch.rand(likely.shape, generator=g, device="cuda"))
    x[:, 1::501] = float("-inf")
    return x.to(DTYPES[case["dtype"]])


def _settings(case, seed):
    rows, f = case["rows"], case["filters"]
    r = np.random.default_rng(seed + 5)

    def tensor(v, dtype):
        return torch.from_numpy(v.astype(dtype)).cuda()

    s = {"u": tensor(r.random(rows, dtype=np.float32), np.float32), "temperature": tensor(r.uniform(0.6, 1.3, rows), np.float32),
         "top_k": None, "top_p": None, "min_p": None}
    if f in ("all", "top_k"):
        s["top_k"] = tensor(r.integers(1, max(2, min(200, case["vocab"])), rows), np.int32)
    if f in ("all", "top_p"):
        s["top_p"] = tensor(r.uniform(0.7, 0.99, rows), np.float32)
    if f in ("all", "min_p"):
        s["min_p"] = tensor(r.uniform(0.0, 0.1, rows), np.float32)
    return s


def prepare(case, seed):
    op = case["op"]
    state = {"case": case}
    if op == "scan_step":
        n = case["tokens"]
        state.update(_scan_inputs(case, seed), pool=_states(case, n + 3, seed), slots=_slots(n, seed))
    elif op in ("scan_chunk", "scan_grad"):
        lens = _lengths(case)
        state.update(_scan_inputs(case, seed), lens=lens, slots=None, initial=None,
                     cu=torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda"))
        if op == "scan_grad":
            if case["initial"]:
                state["initial"] = _states(case, len(lens), seed)
        elif case["initial"]:
            state.update(slots=_slots(len(lens), seed), initial=_states(case, len(lens) + 3, seed))
            state["final"] = state["initial"].clone()
        else:
            state["final"] = torch.zeros(len(lens), case["channels"], case["n"], device="cuda")
    elif op == "quantize":
        state["x"] = _activations(case, seed)
    elif op == "matmul":
        state.update(_product_inputs(case, seed))
    else:
        state.update(_settings(case, seed), logits=_logits(case, seed))
    torch.cuda.synchronize()
    return state


# ---- plain forms ----

def _padded(s, case):
    """The tokens as [T, sequences]: their row in the packed arrays, and whether there is one."""
    if case["op"] == "scan_step":
        at = torch.arange(case["tokens"], device="cuda")[None]
        return at, torch.ones_like(at, dtype=torch.bool)
    at = s["cu"][:-1].long() + torch.arange(max(s["lens"]), device="cuda")[:, None]
    live = at < s["cu"][1:]
    return torch.where(live, at, 0), live


def _terms(s, case, at, live):
    """Of the tokens at [T, N]: s, x [T, N, ch] and B, C [T, N, ch or 1, n] in 32 bits, and the decays e^(s A)."""
    step = torch.nn.functional.softplus(s["dt"][at].float() + s["dt_bias"], threshold=80.0)
    step = torch.where(live[..., None], step, 0.0)      # (a token that is none leaves the state as it is)
    rep = case["channels"] // case["groups"] if case["groups"] > 1 else 1
    b, c = (s[n][at].float().repeat_interleave(rep, 2) for n in ("b", "c"))
    return step, s["x"][at].float(), b, c, torch.exp(step[..., None] * s["a"])


def _plain_scan(s, case, h):
    """The recurrence from the states h [N, ch, n]; returns the outputs at [T, N] of the packed rows, and the last states."""
    at, live = _padded(s, case)
    out = torch.empty_like(s["x"])
    for t0 in range(0, at.shape[0], 64):                # (64 tokens at a time: the decays of all would fill the memory)
        a, l = at[t0:t0 + 64], live[t0:t0 + 64]
        step, x, b, c, decay = _terms(s, case, a, l)
        states = (step * x)[..., None] * b
        for t in range(a.shape[0]):
            h = states[t].addcmul_(decay[t], h)
        y = (states * c).sum(-1) + s["d"] * x
        if s["z"] is not None:
            y = y * torch.nn.functional.silu(s["z"][a].float())
        out[a[l]] = y.to(out.dtype)[l]
    return out, h


def _plain_scan_step(s, case):
    slots = s["slots"].long()
    out, h = _plain_scan(s, case, s["pool"][slots])
    s["pool"][slots] = h
    return {"out": out, "state": s["pool"]}


def _plain_scan_chunk(s, case):
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(len(s["lens"]), device="cuda")
    out, h = _plain_scan(s, case, s["initial"][slots] if s["initial"] is not None else torch.zeros_like(s["final"]))
    s["final"][slots] = h
    return {"out": out, "state": s["final"]}


def _plain_scan_grad(s, case):
    at, live = _padded(s, case)
    T, N = at.shape
    ch, n, groups = case["channels"], case["n"], case["groups"]
    step, x, b, c, decay = _terms(s, case, at, live)
    h0 = s["initial"] if s["initial"] is not None else torch.zeros(N, ch, n, device="cuda")
    states = (step * x)[..., None] * b
    h = h0
    for t in range(T):
        h = states[t].addcmul_(decay[t], h)
    dout = torch.where(live[..., None], s["dout"][at].float(), 0.0)
    dz, dy = None, dout
    if s["z"] is not None:
        z = s["z"][at].float()
        gate = torch.sigmoid(z)
        dy = dout * z * gate
        dz = dout * ((states * c).sum(-1) + s["d"] * x) * gate * (1 + z * (1 - gate))
    dc = (dy[..., None] * states).view(T, N, groups, ch // groups, n).sum(3)
    grads = dy[..., None] * c                           # dL/dh of each token: what its output asks for, and below what comes back
    g = s["dfinal"]
    if g is not None:
        grads[T - 1] += g
    for t in range(T - 1, 0, -1):
        grads[t - 1].addcmul_(decay[t], grads[t])
    back = torch.cat([h0[None], states[:-1]])           # the state before each token
    back *= decay
    dinitial = decay[0] * grads[0]
    db = (grads * (step * x)[..., None]).view(T, N, groups, ch // groups, n).sum(3)
    into = (grads * b).sum(-1)
    back *= grads
    dstep = (back * s["a"]).sum(-1) + into * x
    da = torch.einsum("tncs,tnc->cs", back, step)
    draw_ = dstep * torch.sigmoid(s["dt"][at].float() + s["dt_bias"])
    draw_ = torch.where(live[..., None], draw_, 0.0)

    def rows(v, like):
        r = torch.empty_like(like)
        r[at[live]] = v[live].to(like.dtype)
        return r

    return {"x": rows(step * into + dy * s["d"], s["x"]), "dt": rows(draw_, s["dt"]), "a": da, "b": rows(db, s["b"]), "c": rows(dc, s["c"]),
            "d": (dy * x).sum((0, 1)), "z": None if dz is None else rows(dz, s["z"]), "dt_bias": draw_.sum((0, 1)),
            "initial": dinitial if s["initial"] is not None else None}


def _blocks(x, rows):
    """x padded with zeros to whole blocks, as [row blocks, rows, column blocks, 128]."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def _plain_quantize(s, case):
    x = _blocks(s["x"].float(), case["block_rows"])
    scale = (x.abs().amax((1, 3)).double() / 448.0).float().clamp(min=2.0 ** -126)
    inverse = (1.0 / scale.double()).float()            # a value next to a border of two codes is decided by these 32 bits
    codes = (x * inverse[:, None, :, None]).clamp(-448.0, 448.0).to(F8)
    codes = codes.view(codes.shape[0] * codes.shape[1], -1)[:case["rows"], :case["cols"]].contiguous()
    return {"codes": codes, "scales": scale}


def _plain_matmul(s, case):
    k, n = case["k"], case["n"]
    x = s["x"].float() * s["sx"].repeat_interleave(128, 1)[:, :k]
    w = s["w"].float() * s["sw"].repeat_interleave(128, 1)[:, :k].repeat_interleave(128, 0)[:n]
    y = torch.matmul(x, w.T)
    return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[case["dtype"]])


def _plain_sample(s, case):
    l = s["logits"].double()
    l, order = torch.sort(l, dim=1, descending=True, stable=True)      # (equal ones in the order of their indexes)
    w = torch.exp((l - l[:, :1]) / s["temperature"].double()[:, None])
    w = torch.round(w * ONE).long()
    rank = torch.arange(l.shape[1], device="cuda")
    if s["top_k"] is not None:
        w = torch.where(rank < s["top_k"][:, None], w, 0)
    if s["top_p"] is not None:
        before = w.cumsum(1) - w
        w = torch.where(before.double() < s["top_p"].double()[:, None] * w.sum(1, keepdim=True).double(), w, 0)
    if s["min_p"] is not None:
        w = torch.where(w.double() >= s["min_p"].double()[:, None] * ONE, w, 0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    upto = kept.cumsum(1)
    over = upto.double() > s["u"].double()[:, None] * upto[:, -1:].double()
    return over.to(torch.int8).argmax(1).to(torch.int32)


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"scan_step": _plain_scan_step, "scan_chunk": _plain_scan_chunk, "scan_grad": _plain_scan_grad,
                "quantize": _plain_quantize, "matmul": _plain_matmul, "sample": _plain_sample}[op](s, case)
    from redukt_amd import ops

    if op == "scan_step":
        out = ops.scan_step(s["x"], s["dt"], s["a"], s["b"], s["c"], s["pool"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                            slots=s["slots"])
        return {"out": out, "state": s["pool"]}
    if op == "scan_chunk":
        out = ops.scan_chunk(s["x"], s["dt"], s["a"], s["b"], s["c"], s["cu"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                             state_in=s["initial"], state_out=s["final"], slots=s["slots"])
        return {"out": out, "state": s["final"]}
    if op == "scan_grad":
        g = ops.scan_grad(s["dout"], s["x"], s["dt"], s["a"], s["b"], s["c"], s["cu"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                          state_in=s["initial"], dstate_out=s["dfinal"])
        return {"x": g.x, "dt": g.dt, "a": g.a, "b": g.b, "c": g.c, "d": g.d, "z": g.z, "dt_bias": g.dt_bias, "initial": g.state_in}
    if op == "quantize":
        codes, scales = ops.quantize_blocks(s["x"], block_rows=case["block_rows"])
        return {"codes": codes, "scales": scales}
    if op == "matmul":
        return ops.fp8_matmul(s["x"], s["sx"], s["w"], s["sw"], bias=s["bias"], dtype=DTYPES[case["dtype"]])
    return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


# ---- what a pass cannot do without ----

def work(case):
    op, size = case["op"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if op == "quantize":
        return {"bytes": case["rows"] * case["cols"] * (size + 1) + 4 * -(-case["rows"] // case["block_rows"]) * -(-case["cols"] // 128),
                "flops": 0}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * -(-k // 128) * (m + -(-n // 128)) + 4 * n * case["bias"] + m * n * size, "flops": 2 * m * n * k}
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 0}
    T, ch, n = case["tokens"], case["channels"], case["n"]
    grad = op == "scan_grad"
    wide = (7 if grad else 4) if case["gate"] else (5 if grad else 3)
    state = 4 * case["seqs"] * ch * n * ((3 if grad else 2) if case["initial"] else (0 if grad else 1))
    # a token, channel and n: the decay's factor and power, the input, the state and the output (7 operations); backward again, and
    # the state's gradient, four products with it and their sums
    return {"bytes": T * (ch * wide * size + case["groups"] * n * (4 if grad else 2) * size) + state + (2 if grad else 1) * 4 * ch * (n + 2),
            "flops": (20 if grad else 7) * T * ch * n}


# ---- 64-bit results ----

def _exact_scan(x, case, lens, h0):
    """Outputs and last states in 64 bits, h0 [sequences, channels, n]: a sequence's tokens are joined pair by pair, then
    four by four and so on, each with its span's decay and contribution.  Differentiable."""
    rep = case["channels"] // case["groups"]
    outs, finals, start = [], [], 0
    for i, length in enumerate(lens):
        r = slice(start, start + length)
        raw = x["dt"][r] + x["dt_bias"]
        step = torch.logaddexp(raw, torch.zeros_like(raw))
        decay = torch.exp(step[..., None] * x["a"])
        b, c = (x[k][r].repeat_interleave(rep, 1) for k in ("b", "c"))
        h = (step * x["x"][r])[..., None] * b
        h = torch.cat([h[:1] + decay[:1] * h0[i], h[1:]])
        span = 1
        while span < length:
            h = torch.cat([h[:span], h[span:] + decay[span:] * h[:-span]])
            decay = torch.cat([decay[:span], decay[span:] * decay[:-span]])
            span *= 2
        y = (h * c).sum(-1) + x["d"] * x["x"][r]
        if x["z"] is not None:
            y = y * x["z"][r] * torch.sigmoid(x["z"][r])
        outs.append(y)
        finals.append(h[-1])
        start += length
    return torch.cat(outs), torch.stack(finals)


def _doubles(case, seed):
    return {k: None if v is None else v.double() for k, v in _scan_inputs(case, seed).items()}


def _some_channels(x, case, c0, c1):
    """The inputs of channels c0 to c1, which lie in one group."""
    per = case["channels"] // case["groups"]
    g = c0 // per
    part = {k: v if v is None else v[:, c0:c1] for k, v in x.items() if k in ("x", "dt", "z", "dout", "dfinal")}
    part.update({k: x[k][c0:c1] for k in ("a", "d", "dt_bias")}, **{k: x[k][:, g:g + 1] for k in ("b", "c")})
    return part, g, dict(case, channels=c1 - c0, groups=1)


def _exact_grad(case, seed):
    x, lens = _doubles(case, seed), _lengths(case)
    h0 = (_states(case, len(lens), seed) if case["initial"] else torch.zeros(len(lens), case["channels"], case["n"], device="cuda")).double()
    names = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias")
    got = {k: None if x[k] is None else torch.zeros_like(x[k]) for k in names}
    got["initial"] = torch.zeros_like(h0)
    per = case["channels"] // case["groups"]
    for g in range(case["groups"]):
        for c0 in range(g * per, (g + 1) * per, 128):
            c1 = min(c0 + 128, (g + 1) * per)
            part, _, sub = _some_channels(x, case, c0, c1)
            leaves = {k: part[k].clone().requires_grad_() for k in names if part[k] is not None}
            leaves["initial"] = h0[:, c0:c1].clone().requires_grad_()
            out, final = _exact_scan(dict(part, **leaves), sub, lens, leaves["initial"])
            loss = (out * part["dout"]).sum()
            if part["dfinal"] is not None:
                loss = loss + (final * part["dfinal"]).sum()
            found = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
            for k, v in found.items():
                if k in ("b", "c"):
                    got[k][:, g:g + 1] += v
                elif k in ("a", "d", "dt_bias"):
                    got[k][c0:c1] = v
                else:
                    got[k][:, c0:c1] = v
    if not case["initial"]:
        got["initial"] = None
    return got


def _to_e4m3(r):
    """Values within 448 to the nearest of e4m3's, halves to the even one: steps of 2^(e - 3), e at least -6."""
    e = np.floor(np.log2(np.maximum(np.abs(r), 2.0 ** -40)))
    step = np.exp2(np.maximum(e, -6.0) - 3.0)
    return np.rint(r / step) * step


def exact(case, seed):
    op = case["op"]
    if op == "scan_grad":
        return _exact_grad(case, seed)
    if op in ("scan_step", "scan_chunk"):
        lens = [1] * case["tokens"] if op == "scan_step" else _lengths(case)
        if case["initial"]:
            pool, slots = _states(case, len(lens) + 3, seed).double(), _slots(len(lens), seed).long()
        else:
            pool = torch.zeros(len(lens), case["channels"], case["n"], dtype=torch.float64, device="cuda")
            slots = torch.arange(len(lens), device="cuda")
        x = _doubles(case, seed)
        out = torch.zeros_like(x["x"])
        per = case["channels"] // case["groups"]
        for c0 in range(0, case["channels"], min(per, 512)):
            c1 = min(c0 + min(per, 512), (c0 // per + 1) * per)
            part, _, sub = _some_channels(x, case, c0, c1)
            if op == "scan_step":                       # (all streams side by side)
                step = torch.logaddexp(part["dt"] + part["dt_bias"], torch.zeros_like(part["dt"]))
                h = torch.exp(step[..., None] * part["a"]) * pool[slots, c0:c1] + (step * part["x"])[..., None] * part["b"]
                y = (h * part["c"]).sum(-1) + part["d"] * part["x"]
                out[:, c0:c1] = y if part["z"] is None else y * part["z"] * torch.sigmoid(part["z"])
            else:
                out[:, c0:c1], h = _exact_scan(part, sub, lens, pool[slots, c0:c1])
            pool[slots, c0:c1] = h
        return {"out": out, "state": pool}
    if op == "quantize":
        # the recipe's own roundings to 32 bits are part of what the codes and scales are
        x = _activations(case, seed).double().cpu().numpy()
        rows, cols, per = case["rows"], case["cols"], case["block_rows"]
        codes, scales = np.zeros_like(x), np.zeros((-(-rows // per), -(-cols // 128)))
        for j in range(scales.shape[1]):
            cut = x[:, 128 * j:128 * j + 128]
            top = np.maximum.reduceat(np.abs(cut).max(1), np.arange(0, rows, per))
            scales[:, j] = np.maximum((top / 448.0).astype(np.float32), np.float32(2.0 ** -126))
            inverse = np.repeat((1.0 / scales[:, j]).astype(np.float32).astype(np.float64), per)[:rows]
            r = np.clip((cut * inverse[:, None]).astype(np.float32).astype(np.float64), -448, 448)
            codes[:, 128 * j:128 * j + 128] = _to_e4m3(r)
        return {"codes": torch.from_numpy(codes), "scales": torch.from_numpy(scales)}
    if op == "matmul":
        p = _product_inputs(case, seed)
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for c in range(0, case["k"], 128):
            part = torch.matmul(p["x"][:, c:c + 128].double(), p["w"][:, c:c + 128].double().T)
            y += part * p["sx"][:, c // 128, None].double() * p["sw"][:, c // 128].double().repeat_interleave(128)[:case["n"]]
        return y if p["bias"] is None else y + p["bias"].double()
    # row by row on the host: who is kept, in the order of their values, and whose share of the sum holds the random number
    l, s = _logits(case, seed).double().cpu().numpy(), _settings(case, seed)
    s = {k: None if v is None else v.cpu().numpy() for k, v in s.items()}
    tokens = np.zeros(case["rows"], np.int32)
    for i in range(case["rows"]):
        x = l[i]
        w = np.rint(np.exp((x - x.max()) / np.float64(s["temperature"][i])) * ONE).astype(np.int64)
        near = np.flatnonzero(w)                        # (a weight of zero is never drawn and adds nothing)
        near = near[np.lexsort((near, -x[near]))]
        if s["top_k"] is not None:
            near = near[:s["top_k"][i]]
        if s["top_p"] is not None:
            sums = np.cumsum(w[near])
            need = np.float64(s["top_p"][i]) * np.float64(sums[-1])
            near = near[:1 + np.searchsorted(sums.astype(np.float64), need)]
        if s["min_p"] is not None:
            near = near[w[near] >= np.float64(s["min_p"][i]) * ONE]
        near = np.sort(near)
        sums = np.cumsum(w[near])
        tokens[i] = near[np.searchsorted(sums.astype(np.float64), np.float64(s["u"][i]) * np.float64(sums[-1]), side="right")]
    return torch.from_numpy(tokens)
