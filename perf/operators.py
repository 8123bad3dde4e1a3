"""The operators on caller tensors (redukt_amd.ops): what they are measured on.

Four operators, each with its plain form in elementary torch operations (`own` false) and as
a user calls the framework's kernel (`own` true):

  delta_step   the gated delta rule for one token of each of n streams, the states in a pool
               of slots and updated in place:
                   S' = e^g S + beta k (v - e^g S^T k)^T,   o = scale S'^T q
  delta_chunk  the same rule over whole packed sequences, with initial and final states
  quantize     rows of activations to int8 codes with one scale a row (the framework's int8
               recipe: scale amax / 127, its inverse and the scaled value each in 32 bits,
               halves away from zero)
  matmul       the product of int8 codes with a scale per token and per channel

`listed()` holds cases of each from one token to the largest; `draw()` gives more of the same
ranges.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6      # added to the sum of squares that a normalized key or query is divided by


def listed():
    def step(name, n, hk, hv, dk, dv, dtype, normalize):
        return {"name": name, "op": "delta_step", "n": n, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "dtype": dtype,
                "normalize": normalize}

    def chunk(name, seqs, tokens, hk, hv, dk, dv, dtype, normalize, initial):
        return {"name": name, "op": "delta_chunk", "seqs": seqs, "tokens": tokens, "hk": hk, "hv": hv, "dk": dk,
                "dv": dv, "dtype": dtype, "normalize": normalize, "initial": initial}

    def quantize(name, rows, cols, dtype):
        return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "dtype": dtype}

    def matmul(name, m, n, k, dtype, bias):
        return {"name": name, "op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}

    return [
        # one interactive stream with the heads of RWKV-7 0.1B: latency only
        step("step_1", 1, 12, 12, 64, 64, "bf16", False),
        # a ragged lockstep batch, two value heads to a key head
        step("step_100", 100, 8, 16, 128, 128, "bf16", True),
        # a large serving batch: 2 GB of state read and written
        step("step_500_f32", 500, 16, 32, 128, 128, "f32", True),
        # a short prompt of one stream: less than one chunk
        chunk("chunk_50", 1, 50, 12, 12, 64, 64, "bf16", False, False),
        # a batch of prompts of very different lengths, continued from earlier states
        chunk("chunk_37_ragged", 37, 12000, 8, 16, 128, 128, "bf16", True, True),
        # one long document: little to run side by side
        chunk("chunk_8192", 1, 8192, 16, 32, 128, 128, "bf16", True, False),
        # segments of a few files scored in 32 bits, in the head layout of RWKV-7 0.1B
        chunk("chunk_4_f32", 4, 6001, 12, 12, 64, 64, "f32", False, True),
        # the activations of one token
        quantize("quantize_1", 1, 768, "f32"),
        # the inner activations of a long prompt
        quantize("quantize_8191", 8191, 4096, "bf16"),
        # the head for one stream: the weights are read once
        matmul("matmul_1", 1, 50280, 768, "f32", False),
        # a projection for a ragged lockstep batch
        matmul("matmul_100", 100, 4096, 1536, "bf16", True),
        # a projection for a long prompt: the matrix cores' rate
        matmul("matmul_8192", 8192, 8192, 4096, "bf16", False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    return hk, hk * rng.choice([r for r in (1, 1, 2, 2, 3, 4) if hk * r <= 32]), rng.choice([64, 128]), rng.choice([32, 64, 96, 128, 128, 256])


def draw(rng):
    op = rng.choice(["delta_step", "delta_chunk", "delta_chunk", "quantize", "matmul", "matmul"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "delta_step":
        hk, hv, dk, dv = _heads(rng)
        most = max(1, min(1000, 500 * 32 * 128 * 128 // (hv * dk * dv)))
        return {"op": op, "n": _log_int(rng, 1, most), "hk": hk, "hv": hv, "dk": dk, "dv": dv, "dtype": dtype,
                "normalize": rng.random() < 0.7}
    if op == "delta_chunk":
        hk, hv, dk, dv = _heads(rng)
        most = max(64, min(12000, 8192 * 32 * 128 * 128 // (hv * dk * dv)))
        tokens = _log_int(rng, 1, most)
        return {"op": op, "seqs": _log_int(rng, 1, min(64, tokens)), "tokens": tokens, "hk": hk, "hv": hv, "dk": dk,
                "dv": dv, "dtype": dtype, "normalize": rng.random() < 0.7, "initial": rng.random() < 0.5}
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "cols": rng.choice([64, 200, 768, 1000, 1536, _log_int(rng, 16, 4096)]),
                "dtype": dtype}
    while True:
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 50280), 16 * _log_int(rng, 1, 512)
        if m * n * k <= 8192 * 8192 * 4096 and m * n <= 1 << 27:
            return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}


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


def _rule_inputs(case, tokens, seed):
    """Keys, queries and values as a projection gives them; a decay that forgets over one to
    some hundred tokens, from head to head; write strengths between 0 and 1."""
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q, k = randn(tokens, case["hk"], case["dk"]), randn(tokens, case["hk"], case["dk"])
    if not case["normalize"]:      # the caller has normalized them
        q, k = (x / x.square().sum(-1, keepdim=True).sqrt() for x in (q, k))
    v = randn(tokens, case["hv"], case["dv"])
    rate = torch.exp(randn(1, case["hv"]) - 2.0)
    decay = -rate * torch.nn.functional.softplus(randn(tokens, case["hv"]))
    beta = torch.sigmoid(randn(tokens, case["hv"]))
    return {"q": q.to(dtype), "k": k.to(dtype), "v": v.to(dtype), "g": decay, "beta": beta}


def _states(case, slots, seed):
    g = _generator(seed + 77)
    return 0.3 * torch.randn(slots, case["hv"], case["dk"], case["dv"], generator=g, device="cuda")


def _slots(n, seed):
    """n of the n + 3 slots of a pool, in an order of their own."""
    return torch.from_numpy(np.random.default_rng(seed).permutation(n + 3)[:n].astype(np.int32)).cuda()


def _activations(case, seed):
    """Rows as a norm leaves them, of different magnitudes, a few columns much larger."""
    g = _generator(seed)
    x = torch.randn(case["rows"], case["cols"], generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(case["rows"], 1, generator=g, device="cuda"))
    x[:, :: 97] *= 8.0
    return x.to(DTYPES[case["dtype"]])


def _codes(rows, cols, g):
    """Codes of normally distributed values, the largest of a row about 127."""
    return (torch.randn(rows, cols, generator=g, device="cuda") * 32.0).round().clamp(-127, 127).to(torch.int8)


def _product_inputs(case, seed):
    g = _generator(seed)
    x = {"x": _codes(case["m"], case["k"], g), "w": _codes(case["n"], case["k"], g),
         "sx": torch.exp(0.3 * torch.randn(case["m"], generator=g, device="cuda")) / 32.0,
         "sw": torch.exp(0.3 * torch.randn(case["n"], generator=g, device="cuda")) / (32.0 * case["k"] ** 0.5)}
    x["bias"] = 0.1 * torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
    return x


def prepare(case, seed):
    op = case["op"]
    state = {"case": case}
    if op == "delta_step":
        n = case["n"]
        state.update(_rule_inputs(case, n, seed), pool=_states(case, n + 3, seed), slots=_slots(n, seed))
    elif op == "delta_chunk":
        lens = _lengths(case)
        state.update(_rule_inputs(case, case["tokens"], seed), lens=lens,
                     cu=torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda"))
        if case["initial"]:
            state.update(slots=_slots(len(lens), seed), initial=_states(case, len(lens) + 3, seed))
            state["final"] = state["initial"].clone()
        else:
            state.update(slots=None, initial=None,
                         final=torch.zeros(len(lens), case["hv"], case["dk"], case["dv"], device="cuda"))
    elif op == "quantize":
        state["x"] = _activations(case, seed)
    else:
        state.update(_product_inputs(case, seed))
    torch.cuda.synchronize()
    return state


# ---- plain forms ----

def _unit(x, normalize):
    x = x.float()
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS) if normalize else x


def _rule_step(S, q, k, v, decay, beta):
    """One token of the rule in place on S [B, Dk, Dv]: q, k [B, 1, Dk], v [B, 1, Dv]; decay,
    beta [B, 1, 1].  Returns S'^T q."""
    S *= decay
    S.baddbmm_(k.transpose(1, 2), beta * (v - torch.bmm(k, S)))
    return torch.bmm(q, S)


def _plain_rule(s, case, index, S):
    """The rule over tokens `index` [N, T] of every sequence (-1: none, which leaves the state
    as it is); S [N, Hv, Dk, Dv] becomes the final state.  Returns the outputs [N, T, Hv, Dv]."""
    N, T = index.shape
    hv, dk, dv, group = case["hv"], case["dk"], case["dv"], case["hv"] // case["hk"]
    at, live = index.clamp(min=0), (index >= 0)

    def spread(x, heads, width):        # [tokens, heads, width] -> [T, N Hv, 1, width]
        x = x[at.T].view(T, N, heads, 1, width).expand(T, N, heads, hv // heads, width)
        return x.reshape(T, N * hv, 1, width)

    q = spread(_unit(s["q"], case["normalize"]) * dk ** -0.5, case["hk"], dk)
    k = spread(_unit(s["k"], case["normalize"]), case["hk"], dk)
    v = spread(s["v"].float(), hv, dv)
    decay = torch.where(live[..., None], torch.exp(s["g"])[at], 1.0).transpose(0, 1).reshape(T, N * hv, 1, 1)
    beta = torch.where(live[..., None], s["beta"][at], 0.0).transpose(0, 1).reshape(T, N * hv, 1, 1)
    S = S.view(N * hv, dk, dv)
    out = torch.empty(T, N * hv, 1, dv, device=S.device)
    for t in range(T):
        out[t] = _rule_step(S, q[t], k[t], v[t], decay[t], beta[t])
    return out.view(T, N, hv, dv).transpose(0, 1)


def _plain_delta_step(s, case):
    index = torch.arange(case["n"], device="cuda")[:, None]
    S = s["pool"][s["slots"].long()]
    out = _plain_rule(s, case, index, S)
    s["pool"][s["slots"].long()] = S
    return {"out": out[:, 0].to(s["v"].dtype), "state": s["pool"]}


def _plain_delta_chunk(s, case):
    T = max(s["lens"])
    at = s["cu"][:-1, None].long() + torch.arange(T, device="cuda")
    index = torch.where(at < s["cu"][1:, None], at, -1)
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(len(s["lens"]), device="cuda")
    S = s["initial"][slots] if s["initial"] is not None else torch.zeros_like(s["final"])
    out = _plain_rule(s, case, index, S)
    s["final"][slots] = S
    return {"out": out[index >= 0].to(s["v"].dtype), "state": s["final"]}


def _plain_quantize(s, case):
    x = s["x"].float()
    scale = (x.abs().amax(-1, keepdim=True).double() / 127.0).float()
    scale = torch.where(scale > 0, scale, 1.0)
    r = x * (1.0 / scale.double()).float()          # a value next to a half is decided by these 32 bits
    codes = torch.sign(r) * torch.floor(r.abs().double() + 0.5)
    return {"codes": codes.clamp(-127, 127).to(torch.int8), "scales": scale[:, 0]}


def _plain_matmul(s, case):
    y = torch.matmul(s["x"].double(), s["w"].double().T) * s["sx"].double()[:, None] * s["sw"].double()
    return (y if s["bias"] is None else y + s["bias"].double()).to(DTYPES[case["dtype"]])


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"delta_step": _plain_delta_step, "delta_chunk": _plain_delta_chunk, "quantize": _plain_quantize,
                "matmul": _plain_matmul}[op](s, case)
    from redukt_amd import ops

    if op == "delta_step":
        out = ops.delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["pool"], slots=s["slots"],
                             normalize=case["normalize"])
        return {"out": out, "state": s["pool"]}
    if op == "delta_chunk":
        out = ops.delta_chunk(s["q"], s["k"], s["v"], s["g"], s["beta"], s["cu"], state_in=s["initial"],
                              state_out=s["final"], slots=s["slots"], normalize=case["normalize"])
        return {"out": out, "state": s["final"]}
    if op == "quantize":
        codes, scales = ops.quantize_rows(s["x"])
        return {"codes": codes, "scales": scales}
    return ops.int8_matmul(s["x"], s["sx"], s["w"], s["sw"], bias=s["bias"], dtype=DTYPES[case["dtype"]])


# ---- what a pass cannot do without ----

def work(case):
    op, size = case["op"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if op == "quantize":
        return {"bytes": case["rows"] * (case["cols"] * (size + 1) + 4), "flops": 0}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + 4 * n * case["bias"] + m * n * size, "flops": 2 * m * n * k}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    tokens, streams = (case["n"], case["n"]) if op == "delta_step" else (case["tokens"], case["seqs"])
    state = 4 * hv * dk * dv * (2 if op == "delta_step" or case["initial"] else 1)
    # a token's state is decayed, read for the key, written and read for the query
    return {"bytes": streams * state + tokens * (2 * hk * dk * size + 2 * hv * dv * size + 8 * hv),
            "flops": 6 * tokens * hv * dk * dv}


# ---- 64-bit results ----

def _exact_rule(case, seed, lens, initial):
    """Outputs and final states of sequences of `lens` tokens, 64 at a time: with G the decays'
    running sum, the rows D of a block solve (I + A) D = beta (V - e^G K S), where
    A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i."""
    x = {n: t.double() for n, t in _rule_inputs(case, sum(lens), seed).items()}
    hv, rep, C = case["hv"], case["hv"] // case["hk"], 64
    for n in ("q", "k"):
        if case["normalize"]:
            x[n] = x[n] / torch.sqrt((x[n] ** 2).sum(-1, keepdim=True) + EPS)
        x[n] = x[n].repeat_interleave(rep, 1)
    outs, finals, start = [], [], 0
    eye = torch.eye(C, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        S, rows = initial[i].double(), []
        for c in range(start, start + length, C):
            e = min(c + C, start + length)
            q, k, v = (x[n][c:e].transpose(0, 1) for n in ("q", "k", "v"))
            G, beta = x["g"][c:e].T.cumsum(-1), x["beta"][c:e].T
            D = torch.exp(G[:, :, None] - G[:, None, :]).tril()
            A = (beta[:, :, None] * D * torch.matmul(k, k.transpose(1, 2).contiguous())).tril(-1)
            rhs = beta[:, :, None] * (v - torch.exp(G)[:, :, None] * torch.matmul(k, S))
            d = torch.linalg.solve_triangular(eye[:e - c, :e - c] + A, rhs, upper=False, unitriangular=True)
            o = torch.exp(G)[:, :, None] * torch.matmul(q, S) + torch.matmul(torch.matmul(q, k.transpose(1, 2).contiguous()) * D, d)
            rows.append(o.transpose(0, 1) * case["dk"] ** -0.5)
            left = torch.exp(G[:, -1:] - G)[:, :, None]
            S = torch.exp(G[:, -1])[:, None, None] * S + torch.matmul(k.transpose(1, 2).contiguous(), left * d)
        outs.append(torch.cat(rows))
        finals.append(S)
        start += length
    return torch.cat(outs), torch.stack(finals)


def exact(case, seed):
    op = case["op"]
    if op in ("delta_step", "delta_chunk"):
        lens = [1] * case["n"] if op == "delta_step" else _lengths(case)
        if op == "delta_step" or case["initial"]:
            pool = _states(case, len(lens) + 3, seed).double()
            slots = _slots(len(lens), seed).long()
        else:
            pool = torch.zeros(len(lens), case["hv"], case["dk"], case["dv"], dtype=torch.float64, device="cuda")
            slots = torch.arange(len(lens), device="cuda")
        out, final = _exact_rule(case, seed, lens, pool[slots])
        pool[slots] = final
        return {"out": out, "state": pool}
    if op == "quantize":
        # the recipe's own roundings to 32 bits are part of what the codes and scales are
        x = _activations(case, seed).double().cpu().numpy()
        scale = (np.abs(x).max(-1) / 127.0).astype(np.float32).astype(np.float64)
        scale[scale == 0] = 1.0
        r = (x * (1.0 / scale).astype(np.float32).astype(np.float64)[:, None]).astype(np.float32).astype(np.float64)
        codes = np.clip(np.trunc(r + np.copysign(0.5, r)), -127, 127)
        return {"codes": torch.from_numpy(codes.astype(np.int8)), "scales": torch.from_numpy(scale)}
    p = _product_inputs(case, seed)
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for c in range(0, case["k"], 1024):       # sums of at most 1,024 products are exact in 32 bits
        y += torch.matmul(p["x"][:, c:c + 1024].float(), p["w"][:, c:c + 1024].float().T).double()
    y = y * torch.outer(p["sx"].double(), p["sw"].double())
    return y if p["bias"] is None else y + p["bias"].double()
