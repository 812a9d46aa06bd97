"""W . H(X) with the adapters of many requests, against the definition in 64 bits, in two parts.

Without adapters (every index -1) the result is W . H(X) with H(X) computed in fp32 and rounded to bf16 once: each of its
K terms is off by at most 2^-8 of its size, plus the fp32 error of the transform (log2 K + 1 additions, 2^-24 each of the
row's norm) and of the sum: the tensor cores add 16 products at a time and may cut instead of rounding, 2^-22 of the sizes'
sum for each of the K / 16 additions.

With adapters, the difference from that call (fp32 results: the same transform, the same order of the base's sums, so the
base cancels) is the share sum_r B_mr S_r with S_r = scaling * sum_k A_rk x_k.  Its error:

* S: a sum of K products in fp32, off by at most K units of 2^-24 of the sum of their sizes, however it is ordered (for the
  tensor cores K / 16 additions of 2^-22, the same number); times the scaling, one unit; for prompts rounded to bf16, 2^-8
  of its size;
* B S: rank products (exact in fp32) added to a sum that already holds the base: on the tensor cores rank / 16 + 1
  additions off by at most 2^-22 each of the largest size the sum can have; by fp32 arithmetic (decoding) rank + 2
  additions by 2^-23 each.
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24


def make(N, K, M, R, L, seed=0, spread="runs", device="cuda"):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g) * by).bfloat16().to(device)

    X, W = normal(N, K), normal(M, K, by=K ** -0.5)
    A, B = normal(L, R, K, by=K ** -0.5), normal(L, M, R, by=R ** -0.5)
    scaling = (0.25 + torch.rand(L, generator=g)).to(device)
    if spread == "runs":        # requests of many tokens, one in four without an adapter
        cuts = torch.sort(torch.randint(0, N + 1, (max(1, min(7, N // 3)),), generator=g)).values
        of = torch.randint(-1, L, (len(cuts) + 1,), generator=g)
        index = of[torch.bucketize(torch.arange(N), cuts, right=True)]
    elif spread == "any":       # every token its own, values outside the range among them
        index = torch.randint(-2, L + 2, (N,), generator=g)
    else:
        index = torch.full((N,), int(spread))
    return X, W, A, B, index.int().to(device), scaling


def share64(X, A, B, index, scaling):
    """The adapters' share (tokens, M) in 64 bits, the bound of its error that comes from S in units of its factors, and
    the sum of the sizes of its products."""
    L = A.shape[0]
    X, A, B, index = X.double().cpu(), A.double().cpu(), B.double().cpu(), index.cpu().long()
    sc = torch.ones(L, dtype=torch.float64) if scaling is None else scaling.double().cpu()
    N, M = X.shape[0], B.shape[1]
    out, s_unit, size = (torch.zeros(N, M, dtype=torch.float64) for _ in range(3))
    for a in range(L):
        rows = (index == a).nonzero()[:, 0]
        if len(rows):
            S = X[rows] @ A[a].t() * sc[a]
            out[rows] = S @ B[a].t()
            size[rows] = S.abs() @ B[a].abs().t()
            s_unit[rows] = (X[rows].abs() @ A[a].abs().t() * sc[a].abs()) @ B[a].abs().t()
    return out, s_unit, size


def check_base(base, X, W, signs=None, scale=None):
    """base (tokens, M): the fp32 result without adapters."""
    K = X.shape[1]
    x, w = X.double().cpu(), W.double().cpu()
    if signs is not None:
        x = x * signs.double().cpu()
    h, n = x.clone(), 1
    while n < K:
        h = h.reshape(-1, K // (2 * n), 2, n)
        h = torch.stack([h[:, :, 0] + h[:, :, 1], h[:, :, 0] - h[:, :, 1]], 2).reshape(-1, K)
        n *= 2
    h = h * (K ** -0.5 if scale is None else scale)
    size = h.abs() @ w.abs().t()
    logk = K.bit_length() - 1
    allowed = size * 2.0 ** -8 + (logk + 1) * U * h.norm(dim=1)[:, None] * w.abs().sum(1)[None] * 1.01 + K / 16 * 2.0 ** -22 * size
    off = (base.double().cpu() - h @ w.t()).abs()
    assert bool((off <= allowed).all()), f"off by {float((off - allowed).max()):.3g} too much"


def check_share(got, base, X, A, B, index, scaling, tensor_cores=True):
    """got, base: fp32 results (tokens, M) with and without adapters."""
    want, s_unit, size = share64(X, A, B, index, scaling)
    K, R = X.shape[1], A.shape[1]
    got, base = got.double().cpu(), base.double().cpu()
    allowed = (K + 1) * U * s_unit
    biggest = base.abs() + size * (1 + 2.0 ** -8) + allowed
    if tensor_cores:
        allowed = allowed + size * 2.0 ** -8 + (R // 16 + 2) * 2.0 ** -22 * biggest
    else:
        allowed = allowed + (R + 2) * 2.0 ** -23 * biggest
    off = (got - base - want).abs()
    assert bool((off <= allowed).all()), f"off by {float((off - allowed).max()):.3g} too much"
    none = (index.cpu() < 0) | (index.cpu() >= A.shape[0])
    assert torch.equal(got[none], base[none])   # tokens without an adapter: bit for bit the base


# ---------------------------------------------------------------------------------------------------- without a GPU
def test_refusals_of_the_python_entries(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with pytest.raises(RuntimeError, match="CUDA"):
        X, W, A, B, index, sc = make(4, 64, 32, 8, 2, device="cpu")
        pkg.lora_ht_gemm(X, W, A, B, index)
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(*shape, dtype=dtype, device=device)

        i32, f32 = torch.int32, torch.float32
        good = {"X": t(20, 128), "W": t(48, 128), "A": t(3, 16, 128), "B": t(3, 48, 16), "index": t(20, dtype=i32)}
        bad = [
            {"X": t(20, 128, dtype=f32)}, {"W": t(48, 128, dtype=f32)}, {"A": t(3, 16, 128, dtype=torch.float16)},
            {"X": t(20, 64)}, {"X": t(2, 10, 128)}, {"W": t(48, 128, device="cpu")}, {"index": t(20, dtype=i32, device="cpu")},
            {"A": t(16, 128)}, {"A": t(2, 16, 128)}, {"B": t(3, 47, 16)}, {"B": t(3, 48, 8)}, {"A": t(3, 12, 128), "B": t(3, 48, 12)},
            {"A": t(3, 136, 128), "B": t(3, 48, 136)}, {"A": t(0, 16, 128), "B": t(0, 48, 16)},
            {"A": t(3, 0, 128), "B": t(3, 48, 0)}, {"index": t(20, dtype=torch.int64)}, {"index": t(19, dtype=i32)},
            {"X": t(20, 32), "W": t(48, 32), "A": t(3, 16, 32)}, {"X": t(20, 96), "W": t(48, 96), "A": t(3, 16, 96)},
            {"scaling": t(3)}, {"scaling": t(4, dtype=f32)}, {"out_dtype": torch.float16}, {"out_layout": "tm"},
            {"out": t(20, 48, dtype=f32)}, {"out": t(48, 20)},
        ]
        for change in bad:
            with pytest.raises(RuntimeError):
                pkg.lora_ht_gemm(**{**good, **change})
        del good["X"]
        columns = {"X": t(128, 20), **good}
        for change in ({"X": t(128, 0)}, {"X": t(64, 20)}, {"index": t(3, dtype=i32)}, {"B": t(3, 48, 8)}, {"out": t(20, 48)},
                       {"W": t(48, 128, dtype=f32)}, {"scaling": t(2, dtype=f32)}):
            with pytest.raises(RuntimeError):
                pkg.lora_ht_gemv(**{**columns, **change})


def test_an_output_of_a_graph_is_not_overwritten(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        X, W, A, B, index = t(20, 128), t(48, 128), t(3, 16, 128), t(3, 48, 16), t(20, dtype=torch.int32)
        with pytest.raises(RuntimeError, match="requires grad"):
            pkg.lora_ht_gemm(X, W, A, B, index, out=t(48, 20, dtype=torch.float32).requires_grad_())
        with pytest.raises(RuntimeError, match="requires grad"):
            pkg.lora_ht_gemv(W, t(128, 8), A, B, index[:8], out=t(48, 8, dtype=torch.float32).requires_grad_())


def test_c_entries_refuse_before_the_gpu(lib):
    l = lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255

    def gemm(X=p, W=p, C=p, A=p, B=p, index=p, scaling=p, M=48, N=20, K=128, L=3, R=16, odt=lib.F32, layout=0, signs=None, ws=p,
             nws=1 << 30):
        return l.b200ht_lora_gemm(X, W, C, A, B, index, scaling, M, N, K, L, R, odt, layout, 1.0, signs, ws, nws, None)

    def gemv(X=p, W=p, C=p, A=p, B=p, index=p, scaling=p, M=48, N=20, K=128, L=3, R=16, odt=lib.F32, ws=p, nws=1 << 30):
        return l.b200ht_lora_gemv(W, X, C, A, B, index, scaling, M, K, N, L, R, odt, 1.0, ws, nws, None)

    for f in (gemm, gemv):
        assert f(odt=lib.F16) == -3
        for how in ({"K": 96}, {"K": 32}, {"K": 1 << 16}, {"M": -1}, {"N": -1}, {"L": 0}, {"R": 0}, {"R": 12}, {"R": 136}):
            assert f(**how) == -2, how
        for how in ({"X": None}, {"W": None}, {"C": None}, {"A": None}, {"B": None}, {"index": None}):
            assert f(**how) == -1, how
        for how in ({"X": p + 2}, {"A": p + 8}, {"B": p + 8}, {"C": p + 4}, {"index": p + 2}, {"scaling": p + 2}, {"ws": p + 128}):
            assert f(**how) == -4, how
        assert f(ws=None) == -5 and f(nws=64) == -5
        assert f(M=0, X=None) == 0
    assert gemm(layout=2) == -2 and gemm(signs=p + 2) == -4 and gemm(N=0, X=None) == 0
    assert gemv(N=0) == -2 and gemv(N=65) == -2
    assert l.b200ht_lora_gemm_workspace_bytes(48, 20, 128, 16) >= 20 * 128 * 2 + 20 * 16 * 2
    assert l.b200ht_lora_gemm_workspace_bytes(48, 0, 128, 16) == 0
    assert l.b200ht_lora_gemv_workspace_bytes(48, 128, 20, 16) >= (48 * 20 + 20 * 16) * 4


# --------------------------------------------------------------------------------------------------------- on the GPU
SHAPES = [
    # tokens, K, M, rank, adapters
    (1, 64, 8, 8, 1), (1, 1024, 300, 16, 4), (3, 256, 130, 64, 5), (17, 512, 64, 24, 3), (64, 1024, 96, 128, 2),
    (65, 128, 200, 8, 40), (127, 512, 77, 32, 3), (129, 256, 256, 72, 6), (255, 64, 129, 16, 100), (256, 1024, 384, 64, 4),
    (257, 512, 1, 40, 2), (300, 2048, 130, 120, 9), (1000, 256, 520, 16, 7), (1537, 512, 250, 56, 30), (700, 4096, 64, 128, 3),
    # enough reads of A for the tensor cores' kernel: one K step a CTA, several passes over the adapters, straddled groups
    (1100, 4096, 40, 8, 90), (530, 8192, 72, 24, 25), (2100, 1024, 33, 72, 20), (70, 32768, 16, 120, 9), (9000, 256, 24, 40, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("spread", ["runs", "any"])
@pytest.mark.parametrize("layout", ["mn", "nm"])
def test_prompts(pkg, shape, spread, layout):
    N, K, M, R, L = shape
    X, W, A, B, index, scaling = make(N, K, M, R, L, seed=N, spread=spread)
    base = pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), out_layout=layout)
    got = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout=layout)
    half = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout=layout, out_dtype=torch.bfloat16)
    assert pkg.device_status() == 0
    assert torch.equal(half, got.bfloat16())   # the same sums, rounded once
    if layout == "mn":
        base, got = base.t(), got.t()
    check_base(base, X, W)
    check_share(got, base, X, A, B, index, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("index", ["-1", "0", "2", "7"])
def test_one_adapter_or_none_for_all(pkg, index):
    X, W, A, B, index, _ = make(400, 512, 200, 16, 3, spread=index)
    base = pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), out_layout="nm")
    check_share(pkg.lora_ht_gemm(X, W, A, B, index, out_layout="nm"), base, X, A, B, index, None)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,M,L", [(2560, 64, 4096, 3), (2500, 64, 4090, 200), (1100, 32768, 130, 4), (20000, 2048, 40, 5)])
def test_split_launches_and_chunks(pkg, N, K, M, L):
    """The contraction in two launches (160 tiles of 256 rows on 148 SMs), and tokens in chunks that keep their transform in
    L2: tables, low-rank vectors and rows of B have to move along."""
    X, W, A, B, index, scaling = make(N, K, M, 16, L, seed=5)
    base = pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), out_layout="nm")
    got = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout="nm")
    assert pkg.device_status() == 0
    check_base(base, X, W)
    check_share(got, base, X, A, B, index, scaling)


@pytest.mark.gpu
def test_signs_and_scale_belong_to_the_transform(pkg):
    X, W, A, B, index, scaling = make(270, 512, 140, 32, 4, seed=6)
    signs = torch.randint(0, 2, (512,), generator=torch.Generator().manual_seed(1)).cuda() * 2 - 1
    base = pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), signs=signs, scale=0.5, out_layout="nm")
    check_base(base, X, W, signs, 0.5)
    got = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, signs=signs, scale=0.5, out_layout="nm")
    check_share(got, base, X, A, B, index, scaling)


COLUMNS = [
    # columns, N, M, rank, adapters
    (1, 64, 8, 8, 1), (1, 4096, 1000, 64, 3), (1, 8192, 333, 128, 2), (2, 256, 31, 16, 5), (5, 1024, 130, 24, 2), (16, 4096, 97, 16, 20),
    (13, 512, 65, 72, 4), (8, 8192, 40, 32, 3), (24, 2048, 50, 8, 9), (32, 1024, 70, 120, 5), (64, 128, 33, 64, 6), (3, 32768, 20, 16, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", COLUMNS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("spread", ["any", "0", "-1"])
def test_decoding(pkg, shape, spread):
    columns, N, M, R, L = shape
    X, W, A, B, index, scaling = make(columns, N, M, R, L, seed=columns, spread=spread)
    Xc = X.t().contiguous()
    base = pkg.lora_ht_gemv(W, Xc, A, B, torch.full_like(index, -1))
    got = pkg.lora_ht_gemv(W, Xc, A, B, index, scaling=scaling)
    half = pkg.lora_ht_gemv(W, Xc, A, B, index, scaling=scaling, out_dtype=torch.bfloat16)
    assert pkg.device_status() == 0
    assert torch.equal(half, got.bfloat16())
    if 256 <= N <= 8192:   # beyond, the base is fused_ht_gemv's own (tested with it)
        check_base(base.t(), X, W)
    else:
        assert torch.equal(base, pkg.fused_ht_gemv(W, Xc))
    check_share(got.t(), base.t(), X, A, B, index, scaling, tensor_cores=False)


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [17, 40, 64, 100])
def test_decoding_beyond_one_pass_over_the_weight(pkg, columns):
    X, W, A, B, index, scaling = make(columns, 4096, 100, 16, 6, seed=8, spread="any")
    got = pkg.lora_ht_gemv(W, X.t().contiguous(), A, B, index, scaling=scaling)
    assert got.shape == (100, columns)
    check_share(got.t(), pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), out_layout="nm"), X, A, B, index, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [16384, 32768])
@pytest.mark.parametrize("columns", [4, 5, 17, 64])
def test_decoding_with_long_columns_reads_the_weight_once(pkg, columns, N):
    """The GEMV would read W for every fourth column, or for each: the call has to be the contraction's."""
    X, W, A, B, index, scaling = make(columns, N, 72, 16, 3, seed=columns, spread="any")
    base = pkg.lora_ht_gemv(W, X.t().contiguous(), A, B, torch.full_like(index, -1))
    got = pkg.lora_ht_gemv(W, X.t().contiguous(), A, B, index, scaling=scaling)
    assert got.shape == (72, columns)
    assert torch.equal(got, pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling))
    check_base(base.t(), X, W)
    check_share(got.t(), base.t(), X, A, B, index, scaling)


@pytest.mark.gpu
def test_a_vector_is_one_column(pkg):
    X, W, A, B, index, scaling = make(1, 1024, 50, 8, 2, spread="1")
    assert torch.equal(pkg.lora_ht_gemv(W, X[0], A, B, index), pkg.lora_ht_gemv(W, X.t().contiguous(), A, B, index))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [40, 600])
def test_what_a_token_does_not_own_does_not_reach_it(pkg, N):
    """NaN in the memory of adapters that no token names, and in one token's values, stay where they are."""
    X, W, A, B, index, scaling = make(N, 256, 140, 16, 6, seed=9, spread="any")
    index[index == 3] = 2
    clean = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout="nm")
    A2, B2, sc2, X2 = A.clone(), B.clone(), scaling.clone(), X.clone()
    A2[3], B2[3], sc2[3] = float("nan"), float("inf"), float("nan")
    assert torch.equal(pkg.lora_ht_gemm(X, W, A2, B2, index, scaling=sc2, out_layout="nm"), clean)
    X2[17, 5] = float("nan")
    X2[33, 6] = float("inf")
    got = pkg.lora_ht_gemm(X2, W, A2, B2, index, scaling=sc2, out_layout="nm")
    others = [t for t in range(N) if t not in (17, 33)]
    assert torch.equal(got[others], clean[others]) and torch.isnan(got[17]).all() and not torch.isfinite(got[33]).any()
    Xc = X[:16].t().contiguous()
    clean = pkg.lora_ht_gemv(W, Xc, A, B, index[:16], scaling=scaling)
    assert torch.equal(pkg.lora_ht_gemv(W, Xc, A2, B2, index[:16], scaling=sc2), clean)


@pytest.mark.gpu
def test_views_and_outputs_in_hand(pkg):
    """Strided and oddly aligned inputs are taken (copied where need be); `out` is written in place."""
    X, W, A, B, index, scaling = make(90, 256, 64, 16, 3, seed=10)
    want = pkg.lora_ht_gemm(X, W, A, B, index, out_layout="nm")
    raw = torch.empty(A.numel() + 1, dtype=A.dtype, device="cuda")
    odd = raw[1:].view(A.shape).copy_(A)
    wide = torch.zeros(90, 512, dtype=X.dtype, device="cuda")
    wide[:, 128:384] = X
    every = torch.stack([index, index], 1)[:, 0]
    out = torch.empty(90, 64, device="cuda")
    got = pkg.lora_ht_gemm(wide[:, 128:384], W.t().contiguous().t(), odd, B.transpose(1, 2).contiguous().transpose(1, 2), every,
                           out_layout="nm", out=out)
    assert got is out and torch.equal(got, want)
    assert pkg.lora_ht_gemm(X[:0], W, A, B, index[:0], out_layout="nm").shape == (0, 64)
    with pytest.raises(RuntimeError, match="out has"):
        pkg.lora_ht_gemm(X, W, A, B, index, out_layout="nm", out=torch.empty(64, 90, device="cuda"))


@pytest.mark.gpu
def test_graphs_streams_and_repeats(pkg):
    """Captured twice and replayed side by side on two streams; the same bits on every call."""
    X, W, A, B, index, scaling = make(513, 1024, 320, 32, 12, seed=11, spread="any")
    Xc = X[:16].t().contiguous()

    def call():
        return (pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout="nm", out_dtype=torch.bfloat16),
                pkg.lora_ht_gemv(W, Xc, A, B, index[:16], scaling=scaling))

    want = call()
    for _ in range(3):
        for a, b in zip(call(), want):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(call())
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    assert pkg.device_status() == 0


@pytest.mark.gpu
def test_writes_stay_in_the_result_and_the_workspace(pkg, lib):
    l = lib.load()
    for N, K, M, R, L, layout in ((3, 64, 33, 8, 2, 1), (300, 256, 130, 24, 5, 0), (129, 512, 257, 128, 40, 1)):
        X, W, A, B, index, scaling = make(N, K, M, R, L, seed=12, spread="any")
        n = l.b200ht_lora_gemm_workspace_bytes(M, N, K, R)
        guard = 4096
        ws = torch.full((n + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
        C = torch.full((guard + M * N * 2 + (-M * N * 2) % 256 + guard,), 0xA5, dtype=torch.uint8, device="cuda")
        rc = l.b200ht_lora_gemm(X.data_ptr(), W.data_ptr(), C.data_ptr() + guard, A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                scaling.data_ptr(), M, N, K, L, R, lib.BF16, layout, K ** -0.5, None, ws.data_ptr() + guard, n,
                                torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.error_string(rc)
        want = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout="nm" if layout else "mn", out_dtype=torch.bfloat16)
        assert torch.equal(C[guard:guard + M * N * 2].view(torch.bfloat16), want.view(-1))
        for z in (ws[:guard], ws[guard + n:], C[:guard], C[guard + M * N * 2:]):
            assert bool((z == 0xA5).all())
        if N <= 64:
            n = l.b200ht_lora_gemv_workspace_bytes(M, K, N, R)
            ws = torch.full((n + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
            C.fill_(0xA5)
            Xc = X.t().contiguous()
            rc = l.b200ht_lora_gemv(W.data_ptr(), Xc.data_ptr(), C.data_ptr() + guard, A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                    None, M, K, N, L, R, lib.BF16, K ** -0.5, ws.data_ptr() + guard, n,
                                    torch.cuda.current_stream().cuda_stream)
            assert rc == 0, lib.error_string(rc)
            want = pkg.lora_ht_gemv(W, Xc, A, B, index, out_dtype=torch.bfloat16)
            assert torch.equal(C[guard:guard + M * N * 2].view(torch.bfloat16), want.view(-1))
            for z in (ws[:guard], ws[guard + n:], C[:guard], C[guard + M * N * 2:]):
                assert bool((z == 0xA5).all())


@pytest.mark.gpu
def test_projection_with_adapters_then_norm_and_rotation(pkg):
    """The operators as a layer runs them: one product for queries, keys and values of a prompt, views of it through norm and
    rotation, and the next token of the same requests by the decoding forms, which has to agree with the prompt's."""
    T, K, D, hq, hk, L, R = 70, 1024, 64, 6, 2, 3, 16
    M = (hq + 2 * hk) * D
    X, W, A, B, index, scaling = make(T, K, M, R, L, seed=13)
    g = torch.Generator().manual_seed(14)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).bfloat16().cuda() for _ in range(2))
    pos = torch.arange(T, device="cuda") + 5000
    inv = (1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    qkv = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, out_layout="nm", out_dtype=torch.bfloat16).view(T, -1, D)
    q, k = pkg.norm_rotary_qk(qkv[:, :hq], qkv[:, hq:hq + hk], qw, kw, pos, inv, hadamard=True)
    # the heads' kernel against the definition, on the projection as it came out
    from tests.test_heads import assert_close, forward64
    assert_close(q, forward64(qkv[:, :hq], qw, 1e-6, pos, inv, hadamard=True))
    assert_close(k, forward64(qkv[:, hq:hq + hk], kw, 1e-6, pos, inv, hadamard=True))
    # the last eight tokens again, one call each for all of them
    last = slice(T - 8, T)
    one = pkg.lora_ht_gemv(W, X[last].t().contiguous(), A, B, index[last], scaling=scaling, out_dtype=torch.bfloat16)
    one = one.t().contiguous().view(8, -1, D)
    # Both forms round H(X) to bf16 (at most four times on the way, 2^-8 of the row's norm each), S in one of them, and the
    # result: 2^-8 of |W_m| |x| |H(x)| at most each; the norm and rotation then keep distances relative to the row.
    x64 = X[last].double()
    room = (4 + 4 + 2) * 2.0 ** -8 * (W.double().norm(dim=1)[None] * x64.norm(dim=1)[:, None]).cpu()
    want, s_unit, size = share64(X[last], A, B, index[last], scaling)
    room = room + size * 2.0 ** -7 + qkv[last].double().abs().view(8, M).cpu() * 2.0 ** -7
    assert bool(((one.double() - qkv[last].double()).abs().view(8, M).cpu() <= room).all())
    q1, k1 = pkg.norm_rotary_qk(one[:, :hq], one[:, hq:hq + hk], qw, kw, pos[last], inv, hadamard=True)
    assert_close(q1, forward64(one[:, :hq], qw, 1e-6, pos[last], inv, hadamard=True))
    assert k1.shape == (8, hk, D)


@pytest.mark.gpu
def test_registered_operators(pkg):
    X, W, A, B, index, scaling = make(300, 512, 96, 16, 4, seed=15)
    Xc = X[:8].t().contiguous()
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.b200ht.lora_ht_gemm, (X, W, A, B, index, scaling, 0.5, True, True), test_utils=tests)
    torch.library.opcheck(torch.ops.b200ht.lora_ht_gemm, (X, W, A, B, index, None, 0.5, False, False), test_utils=tests)
    torch.library.opcheck(torch.ops.b200ht.lora_ht_gemv, (W, Xc, A, B, index[:8], scaling, 0.5, False), test_utils=tests)
    want = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling, scale=0.5, out_layout="nm", out_dtype=torch.bfloat16)
    assert torch.equal(torch.ops.b200ht.lora_ht_gemm(X, W, A, B, index, scaling, 0.5, True, True), want)
    with pytest.raises(RuntimeError):   # a serving operator: no gradient
        torch.ops.b200ht.lora_ht_gemm(X.float().bfloat16().requires_grad_(), W, A, B, index, scaling, 0.5, True, False).sum().backward()


@pytest.mark.gpu
def test_another_stream_than_the_current_one_waits_its_turn(pkg):
    """Inputs written on a side stream just before the call on it: every kernel of the chain starts after them."""
    X, W, A, B, index, scaling = make(700, 2048, 512, 32, 9, seed=16, spread="any")
    Xc = X[:8].t().contiguous()
    want = pkg.lora_ht_gemm(X, W, A, B, index, scaling=scaling), pkg.lora_ht_gemv(W, Xc, A, B, index[:8], scaling=scaling)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(10):
            late = [torch.zeros_like(t) for t in (X, W, A, B, index, scaling, Xc)]
            busy = torch.randn(2048, 2048, device="cuda")
            for _ in range(5):
                busy = busy @ busy * 1e-3
            for t, v in zip(late, (X, W, A, B, index, scaling, Xc)):
                t.copy_(v)
            x, w, a, b, i, sc, xc = late
            got = pkg.lora_ht_gemm(x, w, a, b, i, scaling=sc), pkg.lora_ht_gemv(w, xc, a, b, i[:8], scaling=sc)
            for t in late:      # and the inputs may be overwritten right behind the call
                t.zero_()
            assert all(torch.equal(u, v) for u, v in zip(got, want))
    assert pkg.device_status() == 0


@pytest.mark.gpu
def test_results_beyond_32_bits(pkg):
    """More than 2^31 elements of C, the tokens in many chunks' worth of tiles: looked at near its end."""
    N, K, M = 66000, 64, 32768
    g = torch.Generator(device="cuda").manual_seed(17)
    X, W = (torch.randn(n, K, generator=g, device="cuda").bfloat16() for n in (N, M))
    A, B = torch.randn(5, 8, K, generator=g, device="cuda").bfloat16(), torch.randn(5, M, 8, generator=g, device="cuda").bfloat16()
    index = (torch.arange(N, device="cuda") // 300 % 6 - 1).int()
    got = pkg.lora_ht_gemm(X, W, A, B, index, out_layout="nm", out_dtype=torch.bfloat16)
    last = slice(N - 600, N)
    small = pkg.lora_ht_gemm(X[last], W, A, B, index[last], out_layout="nm", out_dtype=torch.float32)
    assert pkg.device_status() == 0
    # The same sums in another order at most: K / 16 + 2 additions of 2^-22 each of the sizes' sum, and the rounding to bf16.
    # S comes from another kernel for so few tokens: both sums are within (K + 1) 2^-24 of the sizes of the true one, and
    # each is rounded to bf16, 2^-8 of its value, so that the two S differ by twice that at most (in the sizes of B S).
    _, s_unit, share = share64(X[last], A, B, index[last], None)
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < K:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    size = share + ((X[last].double().cpu() @ h).abs() / 8) @ W.double().cpu().abs().t()
    room = size * (K / 16 + 2) * 2.0 ** -22 + 2 * (share * 2.0 ** -8 + (K + 1) * U * s_unit)
    want = small.double().cpu()
    off = (got[last].double().cpu() - want).abs()
    assert bool((off <= room + (want.abs() + room) * 2.0 ** -8).all())


BROKEN = [
    # tokens, K, M, rank, adapters, M x N layout, result: the clusters' kernel, tiles of 128 and 256 rows, a tail of 128-row
    # tiles behind 256-row ones, tokens in chunks; the three ways a tile's results leave
    (40, 256, 140, 16, 6, "nm", torch.float32), (40, 256, 130, 16, 6, "mn", torch.bfloat16), (300, 512, 257, 128, 5, "nm", torch.bfloat16),
    (1500, 256, 4096, 72, 7, "mn", torch.float32), (1504, 256, 4096, 24, 7, "mn", torch.bfloat16), (1500, 256, 4096, 8, 7, "nm", torch.bfloat16),
    (2560, 64, 4096, 16, 5, "nm", torch.bfloat16), (2500, 64, 4090, 16, 5, "mn", torch.bfloat16), (3000, 64, 4100, 16, 5, "mn", torch.float32), (1600, 16384, 64, 16, 4, "nm", torch.float32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BROKEN, ids=lambda s: "x".join(map(str, s[:5])) + s[5])
@pytest.mark.parametrize("how", ["all", "one"])
def test_a_broken_adapter_stays_with_its_tokens(pkg, shape, how):
    """Infinities and NaN in an adapter that tokens do use: the others, beside them in every tile, keep their results.

    Both calls have the same H(X) and S, bit for bit.  Where a result is computed again, the two differ by their sums: on the
    tensor cores K / 16 + rank / 16 + 1 additions off by at most 2^-22 each of the sum of the products' sizes; in fp32 K / 8
    + rank / 8 + 3 additions off by 2^-24.  The sizes take the rounding of H(X) and S to bf16 along, 1 + 2^-8."""
    N, K, M, R, L, layout, dtype = shape
    X, W, A, B, index, scaling = make(N, K, M, R, L, seed=21, spread="any")
    index[N // 2:N // 2 + 40] = 1      # whole groups of other adapters, and of the broken one
    index[N // 4:N // 4 + 20] = 2
    broken = B.clone()
    rows = torch.arange(M)
    if how == "all":
        broken[2] = float("inf")
        hit = rows >= 0
    else:
        broken[2, 0, 3] = float("nan")
        broken[2, M - 1, 7] = float("-inf")
        hit = (rows == 0) | (rows == M - 1)

    def call(b, out_dtype):
        y = pkg.lora_ht_gemm(X, W, A, b, index, scaling=scaling, out_layout=layout, out_dtype=out_dtype)
        return (y if layout == "nm" else y.t()).cpu()

    clean, got = call(B, torch.float32), call(broken, torch.float32)
    assert pkg.device_status() == 0
    mine = index.cpu() == 2
    assert torch.equal(got[:, ~hit], clean[:, ~hit])
    assert not torch.isfinite(got[mine][:, hit]).any()
    if how == "one":
        assert torch.isnan(got[mine, 0]).all()
        S = (X[mine.cuda()].double() @ A[2, 7].double() * scaling[2].double()).cpu()
        sure = S.abs() > 1e-3          # the sign of an element far from zero
        assert bool(sure.any()) and torch.equal(got[mine, M - 1][sure], -torch.sign(S[sure]).float() * float("inf"))
    _, _, share = share64(X, A, B, index, scaling)
    x, h, n = X.double().cpu(), X.double().cpu(), 1
    while n < K:
        h = h.reshape(-1, K // (2 * n), 2, n)
        h = torch.stack([h[:, :, 0] + h[:, :, 1], h[:, :, 0] - h[:, :, 1]], 2).reshape(-1, K)
        n *= 2
    size = ((h * K ** -0.5).abs() @ W.double().cpu().abs().t() + share) * (1 + 2.0 ** -8)
    allowed = size * ((K / 16 + R / 16 + 1) * 2.0 ** -22 + (K / 8 + R / 8 + 3) * U)
    off = (got.double() - clean.double()).abs()[~mine]
    assert bool((off <= allowed[~mine]).all())
    if dtype == torch.bfloat16:
        assert torch.equal(call(broken, dtype)[~mine], got.bfloat16()[~mine])
    # a token's own NaN among them
    X[N // 4 + 3, 5] = float("nan")
    again = call(broken, torch.float32)
    assert torch.isnan(again[N // 4 + 3]).all()
    others = ~mine
    others[N // 4 + 3] = False
    assert torch.equal(again[others], got[others])


@pytest.mark.gpu
def test_a_backward_that_saved_an_output_fails_once_it_is_overwritten(pkg):
    X, W, A, B, index, scaling = make(33, 256, 48, 16, 3, seed=22)
    scale = torch.ones(1, device="cuda", requires_grad=True)
    Xc, some = X[:4].t().contiguous(), index[:4].contiguous()
    for shape, call in (((33, 48), lambda out: pkg.lora_ht_gemm(X, W, A, B, index, out_layout="nm", out=out)),
                        ((48, 4), lambda out: pkg.lora_ht_gemv(W, Xc, A, B, some, out=out))):
        out = torch.randn(shape, device="cuda")
        y = (out * scale).sum()
        assert call(out) is out and torch.equal(out, call(torch.empty(shape, device="cuda")))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("entry,columns,K,M,R,L", [
    # the streaming form: clusters of the front kernel, one column, tails of rows, few rows; then more columns than one pass
    ("gemv", 16, 4096, 97, 16, 5), ("gemv", 8, 8192, 333, 128, 3), ("gemv", 1, 256, 1, 8, 1), ("gemv", 31, 1024, 4100, 72, 4),
    ("gemv", 2, 512, 7, 24, 2), ("gemv", 20, 8192, 50, 16, 4), ("gemv", 64, 4096, 40, 16, 4), ("gemv", 5, 32768, 9, 40, 2),
    ("mn", 16, 4096, 97, 16, 5), ("nm", 16, 4096, 97, 16, 5), ("mn", 3, 8192, 130, 120, 2), ("nm", 1, 256, 2000, 8, 3),
    ("nm", 64, 4096, 130, 32, 6), ("mn", 2600, 64, 4090, 8, 40),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_c_entries_write_between_their_guards(pkg, lib, entry, columns, K, M, R, L, dtype):
    """Workspaces and results of just the size asked for, with a pattern on both sides."""
    l = lib.load()
    X, W, A, B, index, scaling = make(columns, K, M, R, L, seed=23, spread="any")
    Xc = X.t().contiguous()
    odt, guard = (lib.F32 if dtype == torch.float32 else lib.BF16), 4096
    nc = M * columns * (4 if dtype == torch.float32 else 2)
    n = l.b200ht_lora_gemv_workspace_bytes(M, K, columns, R) if entry == "gemv" else l.b200ht_lora_gemm_workspace_bytes(M, columns, K, R)
    ws, C = (torch.full((size + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda") for size in (n, nc))
    at = ws.data_ptr() + guard
    assert at % 256 == 0
    stream = torch.cuda.current_stream().cuda_stream
    if entry == "gemv":
        rc = l.b200ht_lora_gemv(W.data_ptr(), Xc.data_ptr(), C.data_ptr() + guard, A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                scaling.data_ptr(), M, K, columns, L, R, odt, K ** -0.5, at, n, stream)
    else:
        rc = l.b200ht_lora_gemm(X.data_ptr(), W.data_ptr(), C.data_ptr() + guard, A.data_ptr(), B.data_ptr(), index.data_ptr(),
                                scaling.data_ptr(), M, columns, K, L, R, odt, lib.OUT_NM if entry == "nm" else lib.OUT_MN, K ** -0.5,
                                None, at, n, stream)
    assert rc == 0, lib.error_string(rc)
    for z in (ws[:guard], ws[guard + n:], C[:guard], C[guard + nc:]):
        assert bool((z == 0xA5).all())
    got = C[guard:guard + nc].view(dtype).view((columns, M) if entry == "nm" else (M, columns))
    want = share64(X, A, B, index, scaling)[0]
    got = (got if entry == "nm" else got.t()).double().cpu()
    # that something was written: far closer to the definition than the results are large (their bounds are tested above)
    base = pkg.lora_ht_gemm(X, W, A, B, torch.full_like(index, -1), out_layout="nm").double().cpu()
    assert float((got - want - base).norm() / (want + base).norm()) <= 2.0 ** -5
    assert pkg.device_status() == 0
