"""Drafting with 4-bit weights and verifying the drafts: the operators' cases, their plain forms and their definition in 64 bits.

A program that drafts with a 4-bit copy of its model quantises the matrices once, multiplies the rows of every step by
them (a row or a few a request while it drafts, many while it reads a prompt, there with the rows in 4 bits too if it
likes), and has the drafts verified against the logits of the model itself.

    kind        quantise: numbers to 4-bit codes with a scale for 32, and to the values that these stand for
                product: rows in 16 or 32 bits times a 4-bit matrix
                both: rows that are quantised, times a 4-bit matrix
                verify: drafted tokens against the model's logits
    rows, k, n  the rows, their width, and the numbers of the result's row (verify: n is the vocabulary)
    dtype, out  the type of the rows and of the result
    epilogue    store, silu (gate rows and up rows of the matrix: silu(gate) * up) or add (into a 32-bit stream)
    bias        whether the matrix comes with one
    requests, drafts, ragged, lookup
                how many requests, how many drafts each has (ragged: from none to twice as many), and whether the drafts
                come from looking text up, with no logits of their own
"""
import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _quantise(name, rows, k, dtype="bfloat16"):
    return {"name": name, "kind": "quantise", "rows": rows, "k": k, "dtype": dtype}


def _product(name, rows, k, n, dtype="bfloat16", out="bfloat16", epilogue="store", bias=False, kind="product"):
    return {"name": name, "kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "out": out, "epilogue": epilogue,
            "bias": bias}


def _verify(name, requests, drafts, n, ragged=False, lookup=False):
    return {"name": name, "kind": "verify", "requests": requests, "drafts": drafts, "n": n, "ragged": ragged,
            "lookup": lookup}


def listed():
    return [
        # the rows of a ragged step, of a width that is not whole blocks
        _quantise("quantise_rows", 77, 2570, "float32"),
        # a gate|up matrix of a large model, as it is loaded
        _quantise("quantise_matrix", 24576, 4096),
        # one request that drafts: the q|k|v matrix
        _product("rows_1", 1, 4096, 6144),
        # eight requests that draft: gate and up with the activation
        _product("rows_8_silu", 8, 4096, 24576, epilogue="silu"),
        # thirty-three requests: the logits of a small model, in 32 bits
        _product("rows_33_logits", 33, 1024, 151936, out="float32"),
        # a prompt of odd length in the 32-bit mode, with biases
        _product("rows_130_float32", 130, 2568, 5120, "float32", "float32", bias=True),
        # a prompt through the largest matrix
        _product("rows_2048", 2048, 4096, 24576),
        # the down matrix with both sides in 4 bits: a few requests, and a long prompt
        _product("both_16", 16, 12288, 4096, kind="both"),
        _product("both_4096", 4096, 12288, 4096, kind="both"),
        # one request with four drafts; a full batch with none to ten drafts each; drafts that were looked up
        _verify("verify_1", 1, 4, 151936),
        _verify("verify_64", 64, 5, 151936, ragged=True),
        _verify("verify_lookup", 16, 3, 32768, ragged=True, lookup=True),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["quantise", "product", "product", "product", "both", "verify"])
    if kind == "quantise":
        rows, k = spread(1, 16384), spread(33, 6000)
        return _without_name(_quantise("", rows, k, rng.choice(["bfloat16", "float32"])))
    if kind == "verify":
        vocabulary = rng.choice([spread(500, 32000), 32768, 151936])
        return _without_name(_verify("", spread(1, 48), rng.randint(1, 6), vocabulary, rng.random() < 0.7,
                                     rng.random() < 0.3))
    rows, k, n = spread(1, 2048), spread(64, 12288), spread(64, 20000)
    if rng.random() < 0.6:
        k = (k + 63) // 64 * 64                  # most widths are whole blocks, as models have them; others are any number
    if rng.random() < 0.6:
        n = (n + 31) // 32 * 32
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"]) if kind == "product" else "bfloat16"
    epilogue = rng.choice(["store", "store", "silu", "add"])
    out = "float32" if epilogue == "add" or rng.random() < 0.3 else dtype
    n += n % 2 if epilogue == "silu" else 0
    return _without_name(_product("", rows, k, n, dtype, out, epilogue, rng.random() < 0.3, kind))


def _without_name(case):
    return {key: v for key, v in case.items() if key != "name"}


def _counts(case):
    """The drafts of every request: given ones, or a walk from none to twice as many."""
    mean, requests = case["drafts"], case["requests"]
    return [(i * 37 + i // 3 + 2) % (2 * mean + 1) if case["ragged"] else mean for i in range(requests)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    if case["kind"] == "verify":
        counts = _counts(case)
        rows, vocabulary = sum(counts) + len(counts), case["n"]
        first = torch.tensor([0] + [n + 1 for n in counts], device="cuda").cumsum(0)
        request = torch.arange(len(counts), device="cuda").repeat_interleave(first.diff())
        drafted = torch.ones(rows, dtype=torch.bool, device="cuda")
        drafted[first[1:] - 1] = False
        logits = normal(rows, vocabulary).mul_(2.5)
        # (requests with temperatures, every fifth of them without: its tokens are the largest logits')
        temperature = 0.5 + torch.rand(len(counts), generator=g, device="cuda")
        temperature[3::5] = 0.0
        t = temperature[request][drafted].unsqueeze(1)
        guess = 0.9 * logits[drafted] + normal(rows - len(counts), vocabulary)
        if case["lookup"]:
            guess = guess + logits[drafted]      # (a text that goes on as the model would, more often than not)
        noise = torch.rand(guess.shape, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
        drawn = torch.where(t > 0, guess / t.clamp(min=0.1) - (-noise.log()).log(), guess).argmax(1)
        state.update(logits=logits, first=first.int(), drafts=drawn.int(), temperature=temperature,
                     draft_logits=None if case["lookup"] else guess,
                     accept_uniform=torch.rand(rows - len(counts), generator=g, device="cuda"),
                     draw_uniform=torch.rand(len(counts), generator=g, device="cuda"))
        return state
    # the rows of a normed stream: most numbers near one, a few columns much larger
    x = normal(case["rows"], case["k"])
    x *= 1.0 + 7.0 * (torch.rand(case["k"], generator=g, device="cuda") < 0.01)
    if case["kind"] == "quantise" and case["rows"] > 4096:
        x *= 0.02                                # a matrix, not rows
    state["x"] = x.to(DTYPES[case["dtype"]])
    if case["kind"] != "quantise":
        codes, scales = [], []
        for part in torch.arange(case["n"], device="cuda").split(16384):
            c, s = _codes(normal(part.numel(), case["k"]).mul_(0.02))
            codes.append(_packed(c))
            scales.append(s)
        state.update(codes=torch.cat(codes), scales=torch.cat(scales))
        state["b"] = normal(case["n"]) if case["bias"] else None
        wide = case["n"] // 2 if case["epilogue"] == "silu" else case["n"]
        state["stream"] = normal(case["rows"], wide) if case["epilogue"] == "add" else None
    return state


# ---- the plain forms -------------------------------------------------------------------------------
def _codes(x):
    """Codes [T, blocks, 32] of 4 bits and scales [T, blocks] (a byte each, 2^(byte - 127)) of the rows of x."""
    T, K = x.shape
    blocks = torch.zeros(T, (K + 31) // 32 * 32, dtype=torch.float32, device=x.device)
    blocks[:, :K] = x
    blocks = blocks.view(T, -1, 32)
    largest = blocks.abs().amax(-1)
    e = (torch.frexp(largest)[1] - 1 - 2).clamp(-127, 127)      # (2^e of the largest number, less the 2 of the largest code)
    e = torch.where(largest > 0, e, torch.full_like(e, -127))
    a = torch.ldexp(blocks.abs(), -e.unsqueeze(-1))
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = code + 8 * torch.signbit(blocks)
    bad = ~torch.isfinite(largest)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    return code, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _packed(code):
    """Two codes a byte, the first in the low half."""
    pairs = code.reshape(code.shape[0], -1, 2)
    return (pairs[..., 0] + 16 * pairs[..., 1]).to(torch.uint8)


def _values(code, scales, K):
    """The numbers that codes and scales stand for, float32 [T, K]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=code.device)
    v = torch.ldexp(grid[code.long()], scales.int().unsqueeze(-1) - 127)
    v = torch.where((scales == 255).unsqueeze(-1), torch.full_like(v, math.nan), v)
    return v.reshape(code.shape[0], -1)[:, :K]


def _unpacked(codes):
    return torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1, 32)


def _plain_product(state):
    w = _values(_unpacked(state["codes"]), state["scales"], state["k"])
    x = state["x"].float()
    if state["kind"] == "both":
        x = _values(*_codes(x), state["k"])
    y = x @ w.T
    if state["b"] is not None:
        y = y + state["b"]
    if state["epilogue"] == "silu":
        gate, up = y.chunk(2, 1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    if state["epilogue"] == "add":
        return state["stream"].add_(y)
    return y.to(DTYPES[state["out"]])


def _weights(logits, t, at):
    """Probabilities in 64 bits of rows at temperature t (0: all on column ``at``)."""
    z = logits.double() / torch.where(t > 0, t, torch.ones_like(t)).double().unsqueeze(1)
    e = torch.exp(z - z.amax(1, keepdim=True))
    e = e / e.sum(1, keepdim=True)
    columns = torch.arange(logits.shape[1], device=logits.device)
    return torch.where((t > 0).unsqueeze(1), e, (columns == at.unsqueeze(1)).double())


def _plain_verify(state):
    logits, first, drafts = state["logits"], state["first"].long(), state["drafts"].long()
    rows, R = logits.shape[0], first.shape[0] - 1
    device = logits.device
    request = torch.searchsorted(first[1:], torch.arange(rows, device=device), right=True)
    t = state["temperature"][request]
    drafted = torch.arange(rows, device=device) != first[request + 1] - 1
    p = _weights(logits, t, logits.argmax(1))
    columns = torch.arange(logits.shape[1], device=device)
    if state["draft_logits"] is None:
        q = (columns == drafts.unsqueeze(1)).double()
    else:
        q = _weights(state["draft_logits"], t[drafted], drafts)
    px = p[drafted].gather(1, drafts.unsqueeze(1)).squeeze(1)
    qx = q.gather(1, drafts.unsqueeze(1)).squeeze(1)
    taken = state["accept_uniform"].double() * qx < px
    number = (torch.arange(rows, device=device) - first[request])
    n = first.diff() - 1
    stop = torch.where(taken, rows, number[drafted])
    accepted = n.scatter_reduce(0, request[drafted], stop, "amin")
    last = first[:-1] + accepted
    w = p[last]
    beside = q[(last - torch.arange(R, device=device)).clamp(max=max(0, q.shape[0] - 1))] if q.shape[0] else torch.zeros_like(w)
    rest = (w - beside).clamp(min=0.0)
    w = torch.where(((accepted < n) & (rest.sum(1) > 0)).unsqueeze(1), rest, w)
    run = w.cumsum(1)
    target = state["draw_uniform"].double() * run[:, -1]
    over = run > target.unsqueeze(1)
    final = (columns * (w > 0)).amax(1)
    token = torch.where(over.any(1), over.int().argmax(1), final)
    out = torch.full((rows,), -1, dtype=torch.int32, device=device)
    out[drafted] = torch.where(number[drafted] < accepted[request[drafted]], state["drafts"], out[drafted])
    out[last] = token.int()
    return {"tokens": out, "accepted": accepted.int()}


# ---- the calls --------------------------------------------------------------------------------------
def _own(state):
    from qwen_engine_amd.kernels import ops

    if state["kind"] == "verify":
        tokens, accepted = ops.verify_drafts(state["logits"], state["first"], state["drafts"], state["draft_logits"],
                                             state["temperature"], state["accept_uniform"], state["draw_uniform"])
        return {"tokens": tokens, "accepted": accepted}
    x = state["x"]
    if state["kind"] == "quantise":
        return ops.mxfp4_values(ops.mxfp4_quantize(x), x.dtype)
    if state["kind"] == "both":
        x = ops.mxfp4_quantize(x)
    epilogue = {"store": ops.EPI_STORE, "silu": ops.EPI_SILU_MUL, "add": ops.EPI_RESIDUAL}[state["epilogue"]]
    return ops.gemm_mxfp4(x, ops.MxFp4(state["codes"], state["scales"], state["k"]), state["b"],
                          out_dtype=DTYPES[state["out"]], out=state["stream"], epilogue=epilogue)


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "verify":
        return _plain_verify(state)
    if state["kind"] == "quantise":
        return _values(*_codes(state["x"]), state["k"]).to(state["x"].dtype)
    return _plain_product(state)


def work(case):
    if case["kind"] == "verify":
        counts = _counts(case)
        rows = sum(counts) + len(counts) + (0 if case["lookup"] else sum(counts))
        return {"bytes": 4.0 * rows * case["n"] + 12.0 * (sum(counts) + 2 * len(counts)), "flops": 4.0 * rows * case["n"]}
    size = {"bfloat16": 2, "float32": 4}
    rows, k = case["rows"], case["k"]
    x, held = rows * k * size[case["dtype"]], 17.0 * ((k + 31) // 32)
    if case["kind"] == "quantise":               # the numbers in, the codes and scales out and in again, the values out
        return {"bytes": 2.0 * x + 2.0 * rows * held, "flops": 8.0 * rows * k}
    wide = case["n"] // 2 if case["epilogue"] == "silu" else case["n"]
    out = rows * wide * (8 if case["epilogue"] == "add" else size[case["out"]])
    return {"bytes": x + case["n"] * held + out + (4 * case["n"] if case["bias"] else 0),
            "flops": 2.0 * rows * k * case["n"]}


# ---- the definition, in 64 bits ---------------------------------------------------------------------
def _nearest(x):
    """The values that the 4-bit form of x stands for, in 64 bits: a number is rounded to a multiple of half its power of
    two (of a half, below one), ties to the even multiple."""
    T, K = x.shape
    blocks = torch.nn.functional.pad(x.double(), (0, -K % 32)).view(T, -1, 32)
    largest = blocks.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.clamp(torch.floor(torch.log2(largest)) - 2, min=-127))
    y = blocks / scale
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs())), min=0.0) - 1)
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0) * scale
    return y.reshape(T, -1)[:, :K]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantise":
        return _nearest(state["x"])
    if case["kind"] == "verify":
        return _exact_verify(state)
    x = state["x"].double()
    if case["kind"] == "both":
        x = _nearest(state["x"])
    nibbles = torch.empty(case["n"], state["codes"].shape[1] * 2, dtype=torch.uint8, device="cuda")
    nibbles[:, 0::2], nibbles[:, 1::2] = state["codes"] % 16, state["codes"] // 16
    sign = 1.0 - 2.0 * (nibbles // 8).double()
    exponent, half = (nibbles // 2 % 4).double(), (nibbles % 2).double()
    w = sign * torch.where(exponent > 0, (1.0 + 0.5 * half) * torch.exp2(exponent - 1), 0.5 * half)
    w = w * torch.exp2(state["scales"].double() - 127.0).repeat_interleave(32, 1)
    y = torch.mm(x, w[:, :case["k"]].T)
    if state["b"] is not None:
        y += state["b"].double()
    if case["epilogue"] == "silu":
        half = case["n"] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    if case["epilogue"] == "add":
        y += state["stream"].double()
    return y


def _exact_verify(state):
    first, drafts = state["first"].tolist(), state["drafts"].tolist()
    tokens, accepted = [], []
    for r, t in enumerate(state["temperature"].tolist()):
        n = first[r + 1] - first[r] - 1
        z = state["logits"][first[r]:first[r + 1]].double()
        mine = drafts[first[r] - r:first[r] - r + n]
        guess = None if state["draft_logits"] is None else state["draft_logits"][first[r] - r:first[r] - r + n].double()
        best = z.argmax(1).tolist()
        j, w = 0, None
        while j < n:
            point = torch.zeros(z.shape[1], dtype=torch.float64, device=z.device)
            if t > 0:
                p = torch.softmax(z[j] / t, 0)
                point[mine[j]] = 1.0
                q = point if guess is None else torch.softmax(guess[j] / t, 0)
                if not float(state["accept_uniform"][first[r] - r + j]) * float(q[mine[j]]) < float(p[mine[j]]):
                    w = torch.relu(p - q)
                    w = w if float(w.sum()) > 0 else p
                    break
            elif mine[j] != best[j]:
                break
            j += 1
        if t > 0:
            run = (torch.softmax(z[n] / t, 0) if w is None else w).cumsum(0)
            token = int((run > float(state["draw_uniform"][r]) * run[-1]).int().argmax())
        else:
            token = best[j]
        tokens += mine[:j] + [token] + [-1] * (n - j)
        accepted.append(j)
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "accepted": torch.tensor(accepted, dtype=torch.int32)}
