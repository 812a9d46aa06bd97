"""Cases for the operators around a rotated projection: positions and norms of queries and keys, and low-rank adapters.

A layer whose weights were folded with a Hadamard matrix computes its projections as W . H(X).  Beside them stand

* ``rotary_qk``       the position rotation of queries and keys, with one or several position axes,
* ``norm_rotary_qk``  the same behind an RMS norm of every head, with its gradients,
* ``lora_ht_gemm`` / ``lora_ht_gemv``  W . H(X) plus the low-rank adapter of each token's request, for prompts and for
  the step that decodes one token of every request.

``own`` chooses between the framework's kernels and the plain form: elementary torch operations in 32 bits (the angles
in 64), rounded once at the end.  ``exact`` computes the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import functools
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = {"short": 1.0e4, "long": 1.0e6}


# --------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------
def _rope(name, op, tokens, q_heads, k_heads, dim, rotary, dtype, sections="", order="blocks", interleaved=False,
          hadamard=False, direction="forward", far=0, packed=True):
    c = {"op": op, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "rotary": rotary,
         "dtype": dtype, "sections": sections, "order": order, "interleaved": interleaved, "hadamard": hadamard,
         "direction": direction, "far": far, "packed": packed}
    return dict(c, name=name) if name else c


def _lora(name, op, tokens, k, m, rank, adapters, requests):
    c = {"op": op, "tokens": tokens, "k": k, "m": m, "rank": rank, "adapters": adapters, "requests": requests}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one conversation, far into a long context: nothing but latency
        _rope("rotary_one_token", "rotary", 1, 32, 8, 128, 128, "bf16", far=1_000_000),
        # a prompt of text and video: three position axes (time, height, width), views of one packed projection
        _rope("rotary_video", "rotary", 4999, 28, 4, 128, 128, "bf16", sections="16,24,24"),
        # the patches of a batch of images in an encoder: two axes, heads of 80, neighbouring pairs, all heads alike
        _rope("rotary_image", "rotary", 9801, 16, 16, 80, 80, "fp16", sections="20,20", interleaved=True),
        # backward of the rotation (with the head rotation that quantised caches use) over a long packed batch
        _rope("rotary_backward", "rotary", 32768, 32, 8, 128, 128, "bf16", hadamard=True, direction="backward",
              packed=False),
        # one token of each of 64 requests at different depths
        _rope("norm_decode", "norm", 64, 32, 8, 128, 128, "bf16", hadamard=True, far=131_072),
        # a prompt, heads rotated for a quantised cache
        _rope("norm_prompt", "norm", 8191, 32, 8, 128, 128, "bf16", hadamard=True),
        # a training step: outputs and the gradients of both inputs and both weights
        _rope("norm_train", "norm", 16384, 16, 8, 128, 128, "bf16", direction="train"),
        # wide heads of which a quarter turns, in full precision, trained
        _rope("norm_train_fp32", "norm", 2047, 16, 2, 256, 64, "fp32", direction="train", packed=False),
        # decoding: 16 requests, each with an adapter of its own, on the square projection of the GEMV benchmark
        _lora("lora_decode_16", "gemv", 16, 4096, 4096, 16, 32, 16),
        # decoding one request on the large weight
        _lora("lora_decode_1", "gemv", 1, 8192, 28672, 64, 8, 1),
        # prompts of eleven requests in one batch, odd number of tokens
        _lora("lora_prompts", "gemm", 2001, 4096, 4096, 32, 32, 11),
        # the headline shape of the benchmark with the prompts of forty requests
        _lora("lora_large", "gemm", 16384, 8192, 28672, 64, 8, 40),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "norm", "norm", "gemv", "gemm"])
    if op in ("rotary", "norm"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2])
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 4, 5, 7])
        tokens = _between(rng, 1, max(64, 30000 * 40 * 128 // ((q_heads + k_heads) * dim * 3)))
        pairs, axes = rotary // 2, rng.choice([1, 1, 2, 3])
        sections, order = "", "blocks"
        if axes == 2:
            a = pairs // 2
            sections = "%d,%d" % (pairs - a, a)
        elif axes == 3:
            a = pairs // 4
            sections, order = "%d,%d,%d" % (pairs - 2 * a, a, a), rng.choice(["blocks", "cycle"])
        hadamard = dim in (64, 128, 256) and rng.random() < 0.4
        return _rope("", op, tokens, q_heads, k_heads, dim, rotary, rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     sections, order, rng.random() < 0.3, hadamard,
                     rng.choice(["forward", "train"] if op == "norm" else ["forward", "backward"]),
                     rng.choice([0, 4096, 131_072, 1_000_000]), rng.random() < 0.6)
    rank = rng.choice([8, 16, 32, 64, 128])
    adapters = _between(rng, 1, 1024 // rank)
    if op == "gemv":
        tokens = _between(rng, 1, 64)
        return _lora("", op, tokens, rng.choice([512, 1024, 2048, 4096, 8192]), _between(rng, 200, 28672), rank, adapters,
                     tokens)
    tokens = _between(rng, 17, 12000)
    return _lora("", op, tokens, rng.choice([512, 1024, 2048, 4096, 8192]), _between(rng, 200, 28672), rank, adapters,
                 _between(rng, 1, min(tokens, 64)))


# --------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------
def _sections(case):
    return tuple(int(v) for v in case["sections"].split(",")) if case["sections"] else None


def _prepare_rope(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    T, hq, hk, D = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # queries and keys as a projection leaves them: some channels are much larger than the others
    gain = torch.exp(0.7 * normal(D))
    if case["packed"]:   # views of one (tokens, (hq + 2 hk) * D) product
        qkv = normal(T, hq + 2 * hk, D).mul_(gain).to(dt)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        q, k = normal(T, hq, D).mul_(gain).to(dt), normal(T, hk, D).mul_(gain).to(dt)
    sections = _sections(case)
    start = int(torch.randint(0, case["far"] + 1, (1,), generator=g, device="cuda")) if case["far"] else 0
    t = torch.arange(T, device="cuda")
    if sections is None:
        if T <= 64 and case["far"]:   # one token of every request
            pos = torch.randint(0, case["far"] + 1, (T,), generator=g, device="cuda")
        else:                         # packed sequences, each counting from its own start
            pos = start + t % max(1, (T + 2) // 3)
    else:                             # frames of a side x side grid
        side = 33
        pos = torch.stack([t // (side * side), t // side % side, t % side][-len(sections):]) + start
    pairs = case["rotary"] // 2
    theta = THETA["long" if case["far"] > 10_000 else "short"]
    inv_freq = (theta ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)).float()
    s = {"case": case, "q": q, "k": k, "positions": pos, "inv_freq": inv_freq, "sections": sections}
    if case["op"] == "norm":
        s["q_weight"] = (1 + 0.2 * normal(D)).to(dt)
        s["k_weight"] = (1 + 0.2 * normal(D)).to(dt)
    if case["direction"] == "train":
        s["dq"], s["dk"] = normal(T, hq, D).to(dt), normal(T, hk, D).to(dt)
    return s


def _prepare_lora(case, seed):
    g = torch.Generator(device="cuda").manual_seed(2000 + seed)
    N, K, M, R, L = case["tokens"], case["k"], case["m"], case["rank"], case["adapters"]

    def normal(*shape, by=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(by).bfloat16()

    W = normal(M, K, by=K ** -0.5)
    A = normal(L, R, K, by=K ** -0.5)
    B = normal(L, M, R, by=0.3 * R ** -0.5)
    scaling = 0.5 + torch.rand(L, generator=g, device="cuda")
    # each request has one of the adapters, or (one in eight) none; its tokens stand next to each other
    n = case["requests"]
    of = torch.randint(0, L, (n,), generator=g, device="cuda")
    of = torch.where(torch.rand(n, generator=g, device="cuda") < 0.125, -1, of)
    if n == N:
        index = of
    else:
        cuts = torch.sort(torch.randint(0, N, (n - 1,), generator=g, device="cuda")).values
        index = of[torch.bucketize(torch.arange(N, device="cuda"), cuts, right=True)]
    if n == 1:
        index = index.clamp(min=0)
    X = normal(K, N) if case["op"] == "gemv" else normal(N, K)
    return {"case": case, "W": W, "X": X, "A": A, "B": B, "index": index.int(), "scaling": scaling}


def prepare(case, seed):
    return _prepare_rope(case, seed) if case["op"] in ("rotary", "norm") else _prepare_lora(case, seed)


# --------------------------------------------------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------------------------------------------------
@functools.cache
def _framework():
    return importlib.import_module("6s894_project_2025_b200")


def _run_own(s):
    ht, c = _framework(), s["case"]
    if c["op"] == "gemm":
        return ht.lora_ht_gemm(s["X"], s["W"], s["A"], s["B"], s["index"], scaling=s["scaling"],
                               out_dtype=torch.bfloat16, out_layout="nm")
    if c["op"] == "gemv":
        return ht.lora_ht_gemv(s["W"], s["X"], s["A"], s["B"], s["index"], scaling=s["scaling"], out_dtype=torch.bfloat16)
    how = {"sections": s["sections"], "axis_order": c["order"], "interleaved": c["interleaved"], "hadamard": c["hadamard"]}
    if c["op"] == "rotary":
        return ht.rotary_qk(s["q"], s["k"], s["positions"], s["inv_freq"], inverse=c["direction"] == "backward", **how)
    out = ht.norm_rotary_qk(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], eps=1e-6, **how)
    if c["direction"] == "train":
        out += ht.norm_rotary_qk_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"],
                                          s["inv_freq"], eps=1e-6, **how)
    return out


# --------------------------------------------------------------------------------------------------------------------
# the plain form
# --------------------------------------------------------------------------------------------------------------------
def _sylvester(n, device):
    """The n x n Hadamard matrix of Sylvester's order: the sign of (i, j) is the parity of the bits of i & j."""
    i = torch.arange(n, device=device)
    v = i[:, None] & i[None, :]
    v = v ^ (v >> 8)
    v = v ^ (v >> 4)
    v = v ^ (v >> 2)
    v = v ^ (v >> 1)
    return 1.0 - 2.0 * (v & 1).float()


def _transform(x):
    """x . H / sqrt(n) along the last dimension: H of a product of two sizes is the product of both along two axes."""
    n = x.shape[-1]
    b = 1 << (n.bit_length() // 2)
    y = x.reshape(-1, n // b, b) @ _sylvester(b, x.device)
    return (_sylvester(n // b, x.device) @ y).reshape(x.shape) * n ** -0.5


def _axis_of_pair(s, pairs):
    """Which position axis turns each pair: blocks of the sections' lengths, or the axes in turn while they last."""
    sections = s["sections"]
    i = torch.arange(pairs, device="cuda")
    if sections is None:
        return torch.zeros_like(i)
    sec = torch.tensor(sections, device="cuda")
    if s["case"]["order"] == "blocks":
        return torch.bucketize(i, torch.cumsum(sec, 0), right=True)
    turn = i % len(sections)
    return torch.where(i < len(sections) * sec[turn], turn, 0)


def _angles(s):
    """cos and sin of every token's pairs, (tokens, 1, pairs)."""
    f = s["inv_freq"].double()
    pos = s["positions"].double()
    pos = pos[None] if pos.dim() == 1 else pos
    a = pos[_axis_of_pair(s, f.shape[0])].t() * f
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    u, rest = x[..., :r], x[..., r:]
    if interleaved:
        a, b = u[..., 0::2], u[..., 1::2]
        u = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = u[..., :r // 2], u[..., r // 2:]
        u = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([u, rest], -1)


def _norm(x, w):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    return x * r * w, r


def _norm_gradients(g, x, w):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    n = x * r
    gw = g * w
    return r * (gw - n * (gw * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))


def _run_rope(s):
    c = s["case"]
    dt, inter, had = DTYPES[c["dtype"]], c["interleaved"], c["hadamard"]
    cos, sin = _angles(s)
    q, k = s["q"].float(), s["k"].float()
    if c["op"] == "rotary" and c["direction"] == "backward":
        q, k = (_transform(q), _transform(k)) if had else (q, k)
        return _turn(q, cos, -sin, inter).to(dt), _turn(k, cos, -sin, inter).to(dt)
    if c["op"] == "norm":
        qw, kw = s["q_weight"].float(), s["k_weight"].float()
        yq, yk = _norm(q, qw)[0], _norm(k, kw)[0]
    else:
        yq, yk = q, k
    yq, yk = _turn(yq, cos, sin, inter), _turn(yk, cos, sin, inter)
    if had:
        yq, yk = _transform(yq), _transform(yk)
    out = (yq.to(dt), yk.to(dt))
    if c["direction"] == "train":
        dq, dk = s["dq"].float(), s["dk"].float()
        if had:
            dq, dk = _transform(dq), _transform(dk)
        dq, dqw = _norm_gradients(_turn(dq, cos, -sin, inter), q, qw)
        dk, dkw = _norm_gradients(_turn(dk, cos, -sin, inter), k, kw)
        out += (dq.to(dt), dk.to(dt), dqw.to(dt), dkw.to(dt))
    return out


def _run_lora(s):
    c = s["case"]
    N, L, R = c["tokens"], c["adapters"], c["rank"]
    X = (s["X"].t() if c["op"] == "gemv" else s["X"]).float()
    y = _transform(X) @ s["W"].float().t()
    # the products with every adapter side by side; each token keeps its own adapter's
    mine = (s["index"][:, None] == torch.arange(L, device="cuda")).float()[:, :, None] * s["scaling"][:, None]
    low = (X @ s["A"].float().reshape(L * R, -1).t()).reshape(N, L, R) * mine
    y = y + low.reshape(N, L * R) @ s["B"].float().transpose(1, 2).reshape(L * R, -1)
    return (y.t().contiguous() if c["op"] == "gemv" else y).bfloat16()


def run(state):
    if own:
        return _run_own(state)
    return _run_rope(state) if state["case"]["op"] in ("rotary", "norm") else _run_lora(state)


# --------------------------------------------------------------------------------------------------------------------
# work and exact values
# --------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("rotary", "norm"):
        D = case["dim"]
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * D
        size = 4 if case["dtype"] == "fp32" else 2
        axes = max(1, len(_sections(case) or ()))
        each = 3 + (5 if case["op"] == "norm" else 0) + (D.bit_length() - 1 if case["hadamard"] else 0)
        passes = 2   # read once, written once
        if case["direction"] == "train":
            passes, each = 2 + 3, 3 * each
        return {"bytes": n * size * passes + case["tokens"] * 8 * axes, "flops": n * each}
    N, K, M, R = case["tokens"], case["k"], case["m"], case["rank"]
    used = min(case["adapters"], case["requests"])
    return {"bytes": 2 * (M * K + N * K + N * M + used * R * (K + M)),
            "flops": 2.0 * N * M * K + 2.0 * N * R * (K + M) + N * K * (K.bit_length() - 1)}


def _butterflies(x):
    """x . H / sqrt(n) in 64 bits, one bit of the index after the other."""
    n, h = x.shape[-1], 1
    y = x.reshape(-1, n).clone()
    while h < n:
        y = y.reshape(-1, n // (2 * h), 2, h)
        y = torch.stack([y[:, :, 0] + y[:, :, 1], y[:, :, 0] - y[:, :, 1]], 2).reshape(-1, n)
        h *= 2
    return y.reshape(x.shape) / math.sqrt(n)


def _exact_rope(case, s):
    T, D, pairs = case["tokens"], case["dim"], case["rotary"] // 2
    pos = s["positions"].reshape(-1, T).double()
    angle = torch.empty(T, pairs, dtype=torch.float64, device="cuda")
    used = [0] * pos.shape[0]
    for i in range(pairs):
        axis = 0
        if s["sections"] is not None:
            if case["order"] == "blocks":
                while sum(s["sections"][:axis + 1]) <= i:
                    axis += 1
            else:
                axis = i % len(s["sections"])
                axis = axis if used[axis] < s["sections"][axis] else 0
        used[axis] += 1
        angle[:, i] = pos[axis] * float(s["inv_freq"][i])
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    at = torch.arange(pairs, device="cuda")
    first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + pairs)

    def rotate(x, t):
        z = torch.complex(x[..., first], x[..., second]) * t
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"y": [], "dx": [], "dw": []}
    for which in ("q", "k"):
        x = s[which].double()
        if case["op"] == "rotary":
            if case["direction"] == "backward":
                out["y"].append(rotate(_butterflies(x) if case["hadamard"] else x, turn.conj()))
            else:
                y = rotate(x, turn)
                out["y"].append(_butterflies(y) if case["hadamard"] else y)
            continue
        w = s[which + "_weight"].double()
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
        y = rotate(x / rms * w, turn)
        out["y"].append(_butterflies(y) if case["hadamard"] else y)
        if case["direction"] == "train":
            g = s["d" + which].double()
            g = rotate(_butterflies(g) if case["hadamard"] else g, turn.conj())
            out["dw"].append((g * x / rms).sum((0, 1)))
            g = g * w
            out["dx"].append(g / rms - x * (g * x).sum(-1, keepdim=True) / (D * rms ** 3))
    return tuple(out["y"] + out["dx"] + out["dw"])


def _exact_lora(case, s):
    X = s["X"].double()
    X = X.t().contiguous() if case["op"] == "gemv" else X
    y = torch.empty(case["tokens"], case["m"], dtype=torch.float64, device="cuda")
    W, H = s["W"].double(), _butterflies(X)
    for t in range(0, case["tokens"], 4096):
        y[t:t + 4096] = H[t:t + 4096] @ W.t()
    for a in range(case["adapters"]):
        rows = (s["index"] == a).nonzero()[:, 0]
        if len(rows):
            low = X[rows] @ s["A"][a].double().t() * s["scaling"][a].double()
            y[rows] += low @ s["B"][a].double().t()
    return y.t().contiguous() if case["op"] == "gemv" else y


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["op"] in ("rotary", "norm") else _exact_lora(case, s)
