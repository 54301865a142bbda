"""Workloads of the training-side dense path: 8-bit activation checkpoints, the matrix product on them, the backward pass that reads
them, and the embedding lookup with its gradient.  `listed()` names the cases, `draw()` makes more of the same ranges, `prepare()` makes a
case's inputs from a seed, `run()` is one pass: with `own` the calls of phonlp_amd.ops, without it the same mathematics in elementary torch
operations.  `exact()` is the definition in 64 bits.

An 8-bit image of a matrix x [M, K] cuts every row into blocks of 128 columns.  A block with the largest finite magnitude a has the
exponent e = the smallest integer >= -126 with a <= 448 * 2^e, and holds the codes e4m3(x * 2^-e), rounded to nearest even.
codes: float8_e4m3fn [M, Kp], Kp = K rounded up to 128, zero behind K; exponents: uint8 e + 127, [M, KB4], KB4 = Kp / 128 rounded up to 4."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the rows of a few sentences kept for the backward pass: a call that is all latency
        {"name": "checkpoint-64x768-bf16", "op": "checkpoint", "M": 64, "K": 768, "type": "bf16"},
        # the input of the parser's first layers, [encoder row ; tag embedding] of 256 sentences of 128 words
        {"name": "checkpoint-32768x868-f32", "op": "checkpoint", "M": 32768, "K": 868, "type": "f32"},
        # one word through the tagger's hidden layer
        {"name": "linear-1x400x768-bf16", "op": "linear", "M": 1, "N": 400, "K": 768, "type": "bf16", "relu": True},
        # the label scorer's bilinear weights (33 relations x 408 columns) on the words of a small, odd batch
        {"name": "linear-2011x13464x408-bf16", "op": "linear", "M": 2011, "N": 13464, "K": 408, "type": "bf16", "relu": False},
        # the three arc scorers' first layers on 256 x 128 words, fp32 in and out
        {"name": "linear-32768x2448x868-f32", "op": "linear", "M": 32768, "N": 2448, "K": 868, "type": "f32", "relu": True},
        # a wide layer at full load: the matrix cores decide
        {"name": "linear-16384x8192x4096-bf16", "op": "linear", "M": 16384, "N": 8192, "K": 4096, "type": "bf16", "relu": False},
        # one sentence's backward pass through the scorers' first layers
        {"name": "backward-31x2448x868-f32", "op": "backward", "M": 31, "N": 2448, "K": 868, "type": "f32", "relu": True},
        # the tagger's hidden layer on an odd number of words, fp32 gradients
        {"name": "backward-8191x400x768-f32", "op": "backward", "M": 8191, "N": 400, "K": 768, "type": "f32", "relu": True},
        # the scorers' first layers on 256 x 128 words, bf16 gradients
        {"name": "backward-32768x2448x868-bf16", "op": "backward", "M": 32768, "N": 2448, "K": 868, "type": "bf16", "relu": True},
        # a sentence's words
        {"name": "embedding-37x64000x768-bf16", "op": "embedding", "N": 37, "V": 64000, "E": 768, "type": "bf16", "scale": 1.0, "spread": "zipf"},
        # tag embeddings: every row of the table's gradient is a sum over a thousand words
        {"name": "embedding-32512x24x100-f32", "op": "embedding", "N": 32512, "V": 24, "E": 100, "type": "f32", "scale": 1.0, "spread": "zipf"},
        # the sub-words of a large batch, scaled by the square root of the width
        {"name": "embedding-65536x64000x768-f32", "op": "embedding", "N": 65536, "V": 64000, "E": 768, "type": "f32", "scale": 27.712812921102035,
         "spread": "zipf"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["checkpoint", "linear", "linear", "backward", "backward", "embedding"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "checkpoint":
        return {"op": op, "M": _log(rng, 1, 32768), "K": _log(rng, 1, 4096), "type": kind}
    if op == "embedding":
        E = _log(rng, 1, 1024)
        return {"op": op, "N": _log(rng, 1, 65536), "V": _log(rng, 2, 64000), "E": E, "type": kind, "scale": rng.choice([1.0, math.sqrt(E)]),
                "spread": rng.choice(["zipf", "even"])}
    most = 16384 * 8192 * 4096 if op == "linear" else 32768 * 2448 * 868
    while True:
        M, N, K = _log(rng, 1, 32768), _log(rng, 8, 13464), _log(rng, 16, 4096)
        if M * N * K <= most and M * N <= 1 << 28:
            return {"op": op, "M": M, "N": N, "K": K, "type": kind, "relu": rng.random() < 0.5}


def work(case):
    s = SIZE[case["type"]]
    if case["op"] == "checkpoint":
        return {"bytes": 2 * case["M"] * case["K"] * s, "flops": 2 * case["M"] * case["K"]}
    if case["op"] == "embedding":
        N, V, E = case["N"], case["V"], case["E"]
        return {"bytes": 8 * N + min(N, V) * E * s + 2 * N * E * s + V * E * s, "flops": 2 * N * E}
    M, N, K = case["M"], case["N"], case["K"]
    kb = -(-K // 128)
    if case["op"] == "linear":
        return {"bytes": M * K * s + N * (K + kb) + 4 * N + M * N * s, "flops": 2 * M * N * K}
    return {"bytes": M * N * s + (M * N // 8 if case["relu"] else 0) + (M + N) * (K + kb) + M * K * s + 4 * N * K + 4 * N, "flops": 4 * M * N * K}


# ---------------------------------------------------------------------------------------------------- plain forms
def _power(e):
    """2^e in fp32 for whole e in -126 .. 127, exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _image(x):
    M, K = x.shape
    blocks = -(-K // 128)
    x = torch.nn.functional.pad(x.float(), (0, blocks * 128 - K)).view(M, blocks, 128)
    fine = torch.isfinite(x)
    a = torch.where(fine, x.abs(), 0.0).amax(2).view(torch.int32)
    e = ((a >> 23) - 135 + ((a & 0x7FFFFF) > 0x600000).int()).clamp(min=-126)
    x = x * _power(-e)[:, :, None]
    x = torch.where((e == 120)[:, :, None], x.clamp(-240.0, 240.0), x)
    codes = torch.where(fine, x, math.nan).to(torch.float8_e4m3fn).view(M, blocks * 128)
    exponents = torch.full((M, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    exponents[:, :blocks] = (e + 127).to(torch.uint8)
    return codes, exponents


def _values(codes, exponents, K):
    M, Kp = codes.shape
    p = _power(exponents[:, : Kp // 128].int() - 127)
    return (codes.float().view(M, Kp // 128, 128) * p[:, :, None]).view(M, Kp)[:, :K]


def _round(x, kind):
    top = torch.finfo(kind).max
    return x.clamp(-top, top).to(kind)


def _pack_bits(mask):
    """Truth values [M, N] -> int32 [M, ceil(N / 32)], column n in bit n % 32 of word n / 32."""
    M, N = mask.shape
    words = -(-N // 32)
    m = torch.nn.functional.pad(mask.long(), (0, words * 32 - N)).view(M, words, 32)
    return (m << torch.arange(32, device=mask.device)).sum(2).to(torch.int32)


def _unpack_bits(bits, N):
    m = (bits[:, :, None] >> torch.arange(32, device=bits.device, dtype=torch.int32)) & 1
    return m.view(bits.shape[0], -1)[:, :N].bool()


# ---------------------------------------------------------------------------------------------------- inputs
def _activations(g, M, K, kind):
    """Rows as an encoder leaves them: normal entries, rows of different loudness, a few loud columns."""
    dev = torch.device("cuda")
    x = torch.randn(M, K, generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device=dev))
    x *= 1.0 + 9.0 * (torch.rand(1, K, generator=g, device=dev) < 0.01)
    return x.to(kind)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    kind = TYPES[case["type"]]
    if case["op"] == "embedding":
        N, V, E = case["N"], case["V"], case["E"]
        u = torch.rand(N, generator=g, device=dev, dtype=torch.float64)
        # "zipf": the rank's frequency falls as 1 / rank; the ranks are spread over the table
        rank = (torch.exp(u * math.log(V + 1.0)) - 1.0) if case["spread"] == "zipf" else u * V
        place = torch.randperm(V, generator=g, device=dev)
        return {"case": case, "table": (0.02 * torch.randn(V, E, generator=g, device=dev)).to(kind),
                "tokens": place[rank.long().clamp(0, V - 1)], "d_out": (1e-3 * torch.randn(N, E, generator=g, device=dev)).to(kind)}
    M, K = case["M"], case["K"]
    x = _activations(g, M, K, kind)
    if case["op"] == "checkpoint":
        return {"case": case, "x": x}
    N = case["N"]
    bound = 1.0 / math.sqrt(K)
    W = (torch.rand(N, K, generator=g, device=dev) * 2.0 - 1.0) * bound
    state = {"case": case, "w": _image(W)}
    if case["op"] == "linear":
        state.update(x=x, bias=(torch.rand(N, generator=g, device=dev) * 2.0 - 1.0) * bound)
        return state
    state["x"] = _image(x)
    state["bits"] = _pack_bits(torch.rand(M, N, generator=g, device=dev) < 0.5) if case["relu"] else None
    state["dy"] = (1e-3 * torch.randn(M, N, generator=g, device=dev)).to(kind)
    return state


# ---------------------------------------------------------------------------------------------------- one pass
def _run_own(s):
    from phonlp_amd import ops

    case = s["case"]
    kind = TYPES[case["type"]]
    if case["op"] == "checkpoint":
        codes, exponents = ops.e4m3_rows(s["x"])
        return ops.e4m3_values(codes, exponents, case["K"], kind)
    if case["op"] == "linear":
        codes, exponents = ops.e4m3_rows(s["x"])
        return ops.linear_e4m3(codes, exponents, s["w"][0], s["w"][1], s["bias"], case["K"], case["relu"], kind)[0]
    if case["op"] == "backward":
        return ops.linear_e4m3_backward(s["dy"], s["bits"], s["x"][0], s["x"][1], s["w"][0], s["w"][1], case["K"])
    out = ops.embedding_rows(s["table"], s["tokens"], case["scale"])
    return out, ops.embedding_rows_grad(s["d_out"], s["tokens"], case["V"], case["scale"])


def _run_plain(s):
    case = s["case"]
    kind = TYPES[case["type"]]
    if case["op"] == "checkpoint":
        return _round(_values(*_image(s["x"]), case["K"]), kind)
    if case["op"] == "linear":
        y = _values(*_image(s["x"]), case["K"]) @ _values(*s["w"], case["K"]).T + s["bias"]
        return (torch.relu(y) if case["relu"] else y).to(kind)
    if case["op"] == "backward":
        dz = s["dy"].float()
        if case["relu"]:
            dz = torch.where(_unpack_bits(s["bits"], case["N"]), dz, 0.0)
        return (dz @ _values(*s["w"], case["K"])).to(kind), dz.T @ _values(*s["x"], case["K"]), dz.sum(0)
    out = (s["table"][s["tokens"]].float() * case["scale"]).to(kind)
    grad = torch.zeros(case["V"], case["E"], device=s["d_out"].device)
    grad.index_add_(0, s["tokens"], s["d_out"].float())
    return out, (grad * case["scale"]).to(kind)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_values(x):
    """The values that an image of x stands for, from the definition."""
    x = x.double()
    M, K = x.shape
    table = torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=x.device)
    power = lambda e: table[e.long() + 200]  # noqa: E731
    out = torch.empty_like(x)
    for k in range(0, K, 128):
        b = x[:, k:k + 128]
        mantissa, e = torch.frexp(b.abs().amax(1))  # a = mantissa * 2^e, 448 = 0.875 * 2^9
        e = (e - 9 + (mantissa > 0.875)).clamp(-126)
        e = torch.where(b.abs().amax(1) == 0, -126, e)[:, None]
        v = b * power(-e)
        v = torch.where(e == 120, v.clamp(-240, 240), v)
        step = power(torch.frexp(v)[1].clamp(min=-5) - 4)  # three bits behind the leading one, steps of 2^-9 below 2^-6
        out[:, k:k + 128] = torch.round(v / step) * step * power(e)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    K = case["K"] if "K" in case else 0
    if case["op"] == "checkpoint":
        return _exact_values(s["x"])
    if case["op"] == "embedding":
        # rows with the same token stand together after a sort; a run's sum is the difference of two running sums
        tokens, order = torch.sort(s["tokens"], stable=True)
        run_sums = torch.nn.functional.pad(torch.cumsum(s["d_out"][order].double(), 0), (0, 0, 1, 0))
        ends = torch.searchsorted(tokens, torch.arange(case["V"] + 1, device=tokens.device))
        seen = torch.nonzero(ends[1:] > ends[:-1])[:, 0]
        grad = torch.zeros(case["V"], case["E"], dtype=torch.float64, device=tokens.device)
        grad[seen] = (run_sums[ends[seen + 1]] - run_sums[ends[seen]]) * case["scale"]
        return s["table"].double()[s["tokens"]] * case["scale"], grad

    def values(image):
        codes, exponents = image
        p = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device=codes.device)[exponents.long()]
        return (codes.to(torch.float64) * p.repeat_interleave(128, 1)[:, : codes.shape[1]])[:, :K]

    w = values(s["w"])
    if case["op"] == "linear":
        y = _exact_values(s["x"]) @ w.T + s["bias"].double()
        return y.clamp(min=0) if case["relu"] else y
    dz = s["dy"].double()
    if case["relu"]:
        n = torch.arange(case["N"], device=dz.device)
        dz = dz * ((s["bits"][:, n // 32] >> (n % 32).int()) & 1)
    return dz @ w, dz.T @ values(s["x"]), dz.sum(0)
