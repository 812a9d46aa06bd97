"""Position rotation of queries and keys, with and without the norm of every head: against the definitions in 64 bits.

Tolerances.  Every result is computed in fp32 and rounded once.  Relative to the 2-norm of its row, in units of 2^-24:
the mean of at most 256 squares and its root 12, the weight 1, the angle 2 (half a unit of 2^-26 turns, times 2 pi) and
cos and sin 4, the rotation 3, the butterflies of H one per bit of the index, 8 at most, their factor 2: 32 in all.  An
orthogonal step does not make an earlier error larger in the 2-norm, and no element is off by more than the 2-norm of
the row's error.  The rounding to the type adds eps / 2 of the value (in fp16 at least half the smallest step, 2^-25).
"""
import ctypes
import math

import pytest
import torch

U = 2.0 ** -24


def axes_of(sections, order, pairs):
    """The axis of every pair, written out."""
    if sections is None:
        return [0] * pairs
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    for i in range(pairs):
        a = i % len(sections)
        a = a if left[a] else 0
        left[a] -= 1
        out.append(a)
    return out


def turn64(x, positions, inv_freq, sections, order, interleaved, inverse=False):
    pairs = inv_freq.numel()
    pos = positions.double().reshape(-1, x.shape[0])
    y = x.clone()
    for i, a in enumerate(axes_of(sections, order, pairs)):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        angle = pos[a] * inv_freq[i].double()
        c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if inverse else 1)
        u, v = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
    return y


def hadamard64(x):
    n = x.shape[-1]
    H = torch.ones(1, 1, dtype=torch.float64)
    while H.shape[0] < n:
        H = torch.cat([torch.cat([H, H], 1), torch.cat([H, -H], 1)])
    return x @ H / math.sqrt(n)


def forward64(x, w, eps, positions, inv_freq, sections=None, order="blocks", interleaved=False, hadamard=False,
              inverse=False):
    x = x.double().cpu()
    positions, inv_freq = positions.cpu(), inv_freq.cpu()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()
    if inverse and hadamard:
        x = hadamard64(x)
    x = turn64(x, positions, inv_freq, sections, order, interleaved, inverse)
    return hadamard64(x) if hadamard and not inverse else x


def assert_close(got, want, units=32, row=None):
    """|got - want| <= eps/2 |want| + units * 2^-24 * (2-norm of the row), element by element."""
    dtype = got.dtype
    got, want = got.double().cpu(), want.cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    near = (want.norm(dim=-1, keepdim=True) if row is None else row) * units * U
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    allowed = torch.finfo(dtype).eps / 2 * (want.abs() + near) + near + tiny
    assert bool((off <= allowed).all()), f"worst {float((off - allowed).max()):.3g} over, at {int((off - allowed).argmax())}"


def make(T, hq, hk, D, pairs, dtype, seed=0, axes=0, packed=False, far=0, pos_dtype=torch.int64, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, hq + 2 * hk, D, generator=g) * torch.exp(torch.randn(D, generator=g))).to(dtype).to(device)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.randint(-far, far + 1, (max(axes, 1), T), generator=g).to(pos_dtype)
    pos = (pos if axes else pos[0]).to(device)
    inv = (1e4 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(device)
    return q, k, pos, inv


# ---------------------------------------------------------------------------------------------------- without a GPU
def test_axis_table(pkg):
    import importlib
    heads = importlib.import_module("6s894_project_2025_b200.heads")
    for sections, order in [((16, 24, 24), "blocks"), ((24, 20, 20), "cycle"), ((4, 2, 2), "cycle"), ((5,), "blocks"),
                            ((0, 3), "blocks"), ((1, 1, 1, 1), "cycle"), ((2, 1), "cycle")]:
        assert list(heads.axis_table(sections, order, sum(sections))) == axes_of(sections, order, sum(sections))
    for sections, order, pairs in [((16, 24), "blocks", 64), ((1, 5), "cycle", 6), ((1,) * 5, "blocks", 5), ((4, -1), "blocks", 3),
                                   ((), "blocks", 0), ((2, 2), "other", 4)]:
        with pytest.raises(RuntimeError):
            heads.axis_table(sections, order, pairs)


def test_refusals_of_the_python_entries(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.rotary_qk(torch.zeros(2, 1, 8), None, torch.arange(2), torch.ones(4))
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(*shape, dtype=dtype, device=device)

        q, k, p, f = t(5, 4, 64), t(5, 2, 64), t(5, dtype=torch.int64), t(32, dtype=torch.float32)
        w = t(64)
        bad = [
            (t(5, 4, 64, dtype=torch.float64), k, p, f, {}), (t(5, 256), k, p, f, {}),
            (t(5, 4, 63), t(5, 2, 63), p, f, {}), (t(5, 4, 258), t(5, 2, 258), p, f, {}),
            (q, t(4, 2, 64), p, f, {}), (q, t(5, 2, 32), p, f, {}), (q, t(5, 2, 64, dtype=torch.float16), p, f, {}),
            (q, t(5, 2, 64, device="cpu"), p, f, {}),
            (q, k, t(4, dtype=torch.int64), f, {}), (q, k, t(5, dtype=torch.float32), f, {}),
            (q, k, t(5, dtype=torch.int64, device="cpu"), f, {}), (q, k, t(1, 5, dtype=torch.int64), f, {}),
            (q, k, p, t(33, dtype=torch.float32), {}), (q, k, p, t(0, dtype=torch.float32), {}), (q, k, p, t(32), {}),
            (q, k, p, f, {"sections": (16, 16)}), (q, k, t(2, 5, dtype=torch.int64), f, {"sections": (16, 15)}),
            (q, k, t(2, 5, dtype=torch.int64), f, {"sections": (16, 16), "axis_order": "turns"}),
            (t(5, 4, 48), t(5, 2, 48), p, t(24, dtype=torch.float32), {"hadamard": True}),
        ]
        for bq, bk, bp, bf, how in bad:
            with pytest.raises(RuntimeError):
                pkg.rotary_qk(bq, bk, bp, bf, **how)
            if bq.dim() == 3 and bq.shape[2] == 64 and bq.dtype == torch.bfloat16:
                with pytest.raises(RuntimeError):
                    pkg.norm_rotary_qk_backward(q, k, bq, bk, w, w, bp, bf, **how)
        for qw, kw in [(t(63), w), (w, t(64, 1)), (w, t(64, dtype=torch.float32)), (t(64, dtype=torch.float16),) * 2,
                       (t(64, device="cpu"), w)]:
            with pytest.raises(RuntimeError):
                pkg.norm_rotary_qk(q, k, qw, kw, p, f)
        with pytest.raises(RuntimeError, match="shapes"):
            pkg.norm_rotary_qk_backward(k, k, q, k, w, w, p, f)
        # in place: strided last dimension, one head shown several times, q and k the same or overlapping heads
        packed = t(5, 8, 64)
        for bq, bk in [(t(5, 64, 4).transpose(1, 2), k), (t(5, 1, 64).expand(5, 4, 64), k), (q, t(1, 2, 64).expand(5, 2, 64))]:
            with pytest.raises(RuntimeError, match="in place|contiguous"):
                pkg.rotary_qk(bq, bk, p, f, inplace=True)
        assert packed.shape == (5, 8, 64)


def test_shared_memory_is_found(pkg):
    import importlib
    heads = importlib.import_module("6s894_project_2025_b200.heads")
    x = torch.zeros(6, 8, 16)
    assert heads._own_memory(x) and heads._own_memory(x[:, 2:5]) and heads._own_memory(x.transpose(0, 1))
    assert not heads._own_memory(x[:, :1].expand(6, 3, 16)) and not heads._own_memory(x[:1].expand(6, 8, 16))
    assert not heads._own_memory(torch.zeros(64).as_strided((4, 3, 8), (8, 4, 1)))
    assert heads._apart(x[:, :4], x[:, 4:6]) and heads._apart(x[:, 6:], x[:, :6]) and heads._apart(x[:3], x[3:])
    assert not heads._apart(x, x) and not heads._apart(x[:, :4], x[:, 3:5]) and not heads._apart(x[:, 3:5], x[:, :4])
    assert not heads._apart(x[:4], x[3:]) and not heads._apart(x[:, :4], x.transpose(0, 1)[:6])


def test_shared_memory_of_one_expanded_token_is_found(pkg):
    """A token's stride may be zero where there is only one."""
    import importlib
    heads = importlib.import_module("6s894_project_2025_b200.heads")
    x = torch.zeros(8, 16).as_strided((1, 8, 16), (0, 16, 1))
    assert heads._apart(x[:, :4], x[:, 4:]) and heads._apart(x[:, 4:], x[:, :4])
    assert not heads._apart(x[:, :4], x[:, 3:]) and not heads._apart(x[:, 3:], x[:, :4])


def test_missing_keys_and_weights_are_named(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        q, k, p, f, w = t(5, 4, 64), t(5, 2, 64), t(5, dtype=torch.int64), t(32, dtype=torch.float32), t(64)
        for bk, qw, kw in [(None, w, None), (k, w, None), (k, None, w), (None, None, None)]:
            with pytest.raises(RuntimeError, match="both weights are required"):
                pkg.norm_rotary_qk(q, bk, qw, kw, p, f)
            with pytest.raises(RuntimeError, match="required"):
                pkg.norm_rotary_qk_backward(q, k, q, bk, qw, kw, p, f)
        for dk, bk in [(None, k), (k, None), (None, None)]:
            with pytest.raises(RuntimeError, match="keys and their gradients"):
                pkg.norm_rotary_qk_backward(q, dk, q, bk, w, w, p, f)


def test_tensors_of_a_graph_are_not_overwritten(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        p, f, w = t(5, dtype=torch.int64), t(32, dtype=torch.float32), t(64)
        q, k, leaf = t(5, 4, 64), t(5, 2, 64), t(5, 6, 64).requires_grad_()
        with torch.no_grad():
            view = leaf[:, :4]
        for bq, bk in [(t(5, 4, 64).requires_grad_(), k), (q, t(5, 2, 64).requires_grad_()), (leaf[:, :4], k), (view, None)]:
            with pytest.raises(RuntimeError, match="requires grad"):
                pkg.rotary_qk(bq, bk, p, f, inplace=True)
        with pytest.raises(RuntimeError, match="requires grad"):
            pkg.norm_rotary_qk(leaf[:, :4], leaf[:, 4:], w, w, p, f, inplace=True)


def test_overwriting_counts_as_a_new_version(pkg):
    import importlib
    ops = importlib.import_module("6s894_project_2025_b200.ops")
    x = torch.zeros(4, 6)
    before = x._version
    ops._overwritten(x[:, :3])
    assert x._version > before and x.detach()._version == x._version
    with torch.inference_mode():
        y = torch.zeros(3)
        ops._overwritten(y)
    ops._overwritten(y)   # an inference tensor has no version, inside the mode or outside


def test_c_entries_refuse_before_the_gpu(lib):
    l = lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) & ~63
    s8, s12 = (ctypes.c_longlong * 8)(), (ctypes.c_longlong * 12)()

    def call(q=p, k=p, qo=p, ko=p, qw=None, kw=None, tokens=1, hq=1, hk=1, D=64, strides=s8, dtype=lib.BF16, pos=p, axes=1,
             table=None, inv=p, pairs=32, flags=0):
        return l.b200ht_rotary_qk(q, k, qo, ko, qw, kw, 1e-6, tokens, hq, hk, D, strides, dtype, pos, 0, 1, axes, table, inv,
                                  pairs, flags, None)

    assert call(dtype=7) == -3
    for how in ({"D": 63}, {"D": 258}, {"D": 0}, {"pairs": 0}, {"pairs": 33}, {"tokens": -1}, {"hq": -1}, {"axes": 0}, {"axes": 5},
                {"axes": 2}, {"axes": 2, "table": bytes([2] * 32)}, {"flags": 64}, {"D": 48, "pairs": 8, "flags": lib.ROT_HADAMARD},
                {"qw": p, "kw": p, "flags": lib.ROT_INVERSE}):
        assert call(**how) == -2, how
    for how in ({"q": None}, {"k": None}, {"qo": None}, {"pos": None}, {"inv": None}, {"strides": None}, {"qw": p}):
        assert call(**how) == -1, how
    for how in ({"q": p + 1}, {"ko": p + 1}, {"q": p + 2, "dtype": lib.F32}, {"pos": p + 2}, {"inv": p + 2},
                {"pos": p + 4, "flags": lib.ROT_POS64}, {"qw": p + 1, "kw": p}, {"qw": p + 2, "kw": p, "flags": lib.ROT_WEIGHT_F32}):
        assert call(**how) == -4, how
    assert call(tokens=0, q=None, pos=None) == 0 and call(hq=0, hk=0, q=None) == 0

    def grad(dq=p, qw=p, dw=p, tokens=1, D=64, flags=0, ws=p, nws=None, strides=s12):
        need = l.b200ht_norm_rotary_qk_backward_workspace_bytes(64)
        return l.b200ht_norm_rotary_qk_backward(dq, p, p, p, qw, p, 1e-6, p, p, dw, p, tokens, 1, 1, D, strides, lib.BF16, p, 0, 1,
                                                1, None, p, 32, flags, ws, need if nws is None else nws, None)

    assert l.b200ht_norm_rotary_qk_backward_workspace_bytes(64) > 0
    assert l.b200ht_norm_rotary_qk_backward_workspace_bytes(300) == 0
    assert grad(D=300) == -2 and grad(flags=lib.ROT_INVERSE) == -2
    assert grad(dq=None) == -1 and grad(qw=None) == -1 and grad(dw=None) == -1 and grad(strides=None) == -1
    assert grad(ws=None) == -5 and grad(nws=64) == -5 and grad(ws=p + 8) == -4


@pytest.mark.parametrize("how", [{"tokens": 1 << 30}, {"tokens": (1 << 31) - 1}, {"hq": 1 << 30}, {"hk": (1 << 31) - 1}])
def test_more_rows_than_32_bits_count_are_refused(lib, how):
    """Tokens rounded up to a block's share, and the heads of both tensors, stay below 2^31."""
    l = lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) & ~63
    a = {"tokens": 1, "hq": 1, "hk": 1} | how
    s8, s12 = (ctypes.c_longlong * 8)(), (ctypes.c_longlong * 12)()
    assert l.b200ht_rotary_qk(p, p, p, p, None, None, 1e-6, a["tokens"], a["hq"], a["hk"], 64, s8, lib.BF16, p, 0, 1, 1, None, p, 32,
                              0, None) == -2
    assert l.b200ht_norm_rotary_qk_backward(p, p, p, p, p, p, 1e-6, p, p, p, p, a["tokens"], a["hq"], a["hk"], 64, s12, lib.BF16, p,
                                            0, 1, 1, None, p, 32, 0, p, 1 << 30, None) == -2


# --------------------------------------------------------------------------------------------------------- on the GPU
SHAPES = [
    # T, q heads, k heads, D, pairs
    (1, 1, 1, 2, 1), (1, 32, 8, 128, 64), (3, 5, 1, 64, 32), (17, 28, 4, 128, 64), (2, 3, 3, 80, 40), (7, 4, 2, 96, 48),
    (5, 2, 1, 256, 32), (4, 16, 2, 256, 128), (9, 3, 2, 128, 32), (3, 2, 2, 36, 18), (6, 7, 1, 66, 20), (33, 1, 0, 64, 32),
    (130, 9, 3, 128, 60), (5, 2, 2, 112, 24), (70, 6, 6, 32, 16), (19, 5, 5, 16, 8),
    # enough tokens that a block takes several of them, with heads that leave some of its groups idle
    (301, 28, 4, 128, 64), (333, 5, 3, 64, 32), (310, 3, 1, 256, 128), (401, 16, 16, 80, 40), (299, 1, 7, 96, 24),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_rotation(pkg, shape, dtype, interleaved, packed):
    T, hq, hk, D, pairs = shape
    q, k, pos, inv = make(T, hq, hk, D, pairs, dtype, packed=packed, far=5000)
    for hadamard in (False, True) if D & (D - 1) == 0 else (False,):
        for inverse in (False, True):
            how = {"interleaved": interleaved, "hadamard": hadamard, "inverse": inverse}
            yq, yk = pkg.rotary_qk(q, k, pos, inv, **how)
            assert yq.dtype == dtype and yq.is_contiguous()
            assert_close(yq, forward64(q, None, 0, pos, inv, **how))
            assert_close(yk, forward64(k, None, 0, pos, inv, **how))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("w_f32", [False, True])
def test_norm_and_its_gradients(pkg, shape, dtype, interleaved, w_f32):
    T, hq, hk, D, pairs = shape
    q, k, pos, inv = make(T, hq, hk, D, pairs, dtype, seed=1, packed=True, far=100)
    g = torch.Generator().manual_seed(2)
    wt = torch.float32 if w_f32 else dtype
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wt).cuda() for _ in range(2))
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    for hadamard in (False, True) if D & (D - 1) == 0 else (False,):
        how = {"interleaved": interleaved, "hadamard": hadamard}
        yq, yk = pkg.norm_rotary_qk(q, k, qw, kw, pos, inv, eps=1e-5, **how)
        gq, gk, gqw, gkw = pkg.norm_rotary_qk_backward(dq, dk, q, k, qw, kw, pos, inv, eps=1e-5, **how)
        for x, w, y, dy, dx, dw in ((q, qw, yq, dq, gq, gqw), (k, kw, yk, dk, gk, gkw)):
            assert_close(y, forward64(x, w, 1e-5, pos, inv, **how))
            gr = forward64(dy, None, 0, pos, inv, inverse=True, **how)
            x64, w64 = x.double().cpu(), w.double().cpu()
            r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + 1e-5)
            h, gw = x64 * r, gr * w64
            # dx: two terms, neither longer than r |g w|, each with the 32 units of its row and the 14 of r and the mean
            # (the gradient's error is relative to |g|, hence the largest weight)
            size = r * (gr.norm(dim=-1, keepdim=True) * w64.abs().max())
            assert_close(dx, r * (gw - h * (gw * h).mean(-1, keepdim=True)), units=128, row=size)
            # dw: 46 units of |row of g| |h_i| a term, and a sum of T * heads terms adds one unit of the terms' sizes each
            rows = x.shape[0] * x.shape[1]
            terms = (gr.norm(dim=-1, keepdim=True) * h.abs()).sum((0, 1))
            assert_close(dw, (gr * h).sum((0, 1)), units=46 + rows, row=terms)
            assert dw.dtype == wt


@pytest.mark.gpu
@pytest.mark.parametrize("sections,order", [((16, 24, 24), "blocks"), ((24, 20, 20), "cycle"), ((32, 32), "blocks"),
                                            ((64,), "blocks"), ((22, 14, 14, 14), "cycle"), ((0, 60, 4), "blocks")])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_several_position_axes(pkg, sections, order, pos_dtype):
    q, k, pos, inv = make(37, 6, 2, 128, 64, torch.bfloat16, axes=len(sections), far=300, pos_dtype=pos_dtype)
    # positions of the tokens next to each other, and of the axes next to each other
    for p in (pos, pos.t().contiguous().t()):
        yq, yk = pkg.rotary_qk(q, k, p, inv, sections=sections, axis_order=order)
        assert_close(yq, forward64(q, None, 0, pos, inv, sections, order))
        assert_close(yk, forward64(k, None, 0, pos, inv, sections, order))


@pytest.mark.gpu
def test_far_positions_keep_their_angle(pkg):
    """A position near 2^31 times a frequency is good to 2^-21 turns, 2 pi * 8 units, added to the 32 of any row."""
    q, k, _, inv = make(64, 4, 1, 128, 64, torch.float32, seed=3)
    pos = torch.tensor([0, 1, -1, 1_000_003, 131_071, -7_777_777, 2 ** 31 - 1, -2 ** 31] * 8, device="cuda")
    for p in (pos, pos.int()):
        yq, _ = pkg.rotary_qk(q, k, p, inv)
        assert_close(yq, forward64(q, None, 0, pos, inv), units=32 + 51)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 66])
def test_in_place_on_views_of_one_projection(pkg, D):
    q, k, pos, inv = make(21, 6, 2, D, D // 2, torch.bfloat16, packed=True, far=50)
    packed = q._base
    before = packed.clone()
    want = pkg.rotary_qk(q, k, pos, inv)
    got = pkg.rotary_qk(q, k, pos, inv, inplace=True)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(packed[:, 8:], before[:, 8:])   # the values of the packed projection stay
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.rotary_qk(q, q, pos, inv, inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.rotary_qk(packed[:, :4], packed[:, 3:5], pos, inv, inplace=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D,pairs", [(128, 64), (64, 32), (256, 32), (80, 40)])
def test_strides_and_alignment_of_any_kind(pkg, D, pairs):
    """Head-major storage, an odd storage offset, a broadcast head, a transposed last dimension, no keys."""
    q, k, pos, inv = make(23, 4, 2, D, pairs, torch.bfloat16, far=70)
    want = pkg.rotary_qk(q, k, pos, inv)
    head_major = q.transpose(0, 1).contiguous().transpose(0, 1)
    raw = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    odd = raw[1:].view(q.shape).copy_(q)
    last = q.transpose(1, 2).contiguous().transpose(1, 2)
    for other in (head_major, odd, last):
        got = pkg.rotary_qk(other, k, pos, inv)
        for a, b in zip(got, want):   # another kernel may round another way: both are near the definition
            assert_close(a, forward64(q if b is want[0] else k, None, 0, pos, inv))
    one = q[:, :1].expand(23, 5, D)
    assert_close(pkg.rotary_qk(one, None, pos, inv)[0], forward64(one, None, 0, pos, inv))
    assert pkg.rotary_qk(q, None, pos, inv)[1] is None
    everywhere = pos[:1].expand(23)
    assert_close(pkg.rotary_qk(q, None, everywhere, inv)[0], forward64(q, None, 0, everywhere, inv))


@pytest.mark.gpu
def test_no_tokens_and_no_heads(pkg):
    q, k, pos, inv = make(0, 4, 2, 64, 32, torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    yq, yk = pkg.norm_rotary_qk(q, k, w, w, pos, inv)
    assert yq.shape == (0, 4, 64) and yk.shape == (0, 2, 64)
    grads = pkg.norm_rotary_qk_backward(q, k, q, k, w, w, pos, inv)
    assert grads[0].shape == (0, 4, 64) and not grads[2].any() and not grads[3].any()
    q, k, pos, inv = make(5, 4, 0, 64, 32, torch.bfloat16)
    grads = pkg.norm_rotary_qk_backward(q, k, q, k, w, w, pos, inv)
    assert grads[2].any() and not grads[3].any()


@pytest.mark.gpu
def test_rows_of_zeros_and_of_not_a_number(pkg):
    """A padded token's row of zeros stays zero (eps keeps the norm finite); NaN and infinity stay in their own row."""
    q, k, pos, inv = make(12, 4, 2, 128, 64, torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    clean = pkg.norm_rotary_qk(q, k, w, w, pos, inv, hadamard=True)[0]
    q2 = q.clone()
    q2[3] = 0
    q2[5, 2, 7] = float("nan")
    q2[6, 1, 9] = float("inf")
    y = pkg.norm_rotary_qk(q2, k, w, w, pos, inv, hadamard=True)[0]
    assert not y[3].any() and torch.isnan(y[5, 2]).all() and not torch.isfinite(y[6, 1]).all()
    for t, h in ((5, 0), (5, 3), (6, 0), (4, 2), (7, 1)):
        assert torch.equal(y[t, h], clean[t, h])
    g = torch.ones_like(q)
    dx = pkg.norm_rotary_qk_backward(g, k, q2, k, w, w, pos, inv)[0]
    assert torch.isfinite(dx[3]).all() and torch.isnan(dx[5, 2]).all() and torch.isfinite(dx[5, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,pairs", [(128, 32), (128, 30), (96, 24), (64, 8), (256, 64), (80, 20), (66, 20), (16, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_dimensions_behind_the_pairs_are_left_alone(pkg, D, pairs, dtype, interleaved):
    """Infinities, NaN and the sign of a zero among them stay, and do not reach the other dimensions."""
    q, k, pos, inv = make(40, 5, 2, D, pairs, dtype, seed=6, far=300)
    clean = pkg.rotary_qk(q, None, pos, inv, interleaved=interleaved)[0]
    for t, value in enumerate([float("inf"), float("-inf"), float("nan"), -0.0] * 8):
        for h in range(5):
            q[t, h, 2 * pairs + (t * 5 + h) % (D - 2 * pairs)] = value
    for inverse in (False, True):
        y = pkg.rotary_qk(q, None, pos, inv, interleaved=interleaved, inverse=inverse)[0]
        # NaN stays NaN, with the payload that the conversion to the type gives every NaN; all else keeps its bits
        whole = torch.int16 if dtype == torch.bfloat16 else torch.int32
        got, want = y[..., 2 * pairs:], q[..., 2 * pairs:]
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got.view(whole)[~nan], want.view(whole)[~nan])
        assert torch.isfinite(y[..., :2 * pairs]).all()
    assert torch.equal(pkg.rotary_qk(q, None, pos, inv, interleaved=interleaved)[0][..., :2 * pairs], clean[..., :2 * pairs])
    # the weights' gradient is a sum over rows for each dimension: an infinite gradient stays in its own
    w = torch.ones(D, dtype=dtype, device="cuda")
    x, dy = torch.ones_like(q), torch.ones_like(q)
    dy[3, 1, D - 1] = float("inf")
    dw = pkg.norm_rotary_qk_backward(dy, dy[:, :0], x, x[:, :0], w, w, pos, inv, interleaved=interleaved)[2]
    assert torch.isinf(dw[D - 1]) and torch.isfinite(dw[:D - 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["rotary", "norm"])
def test_gradients_of_the_registered_operators(pkg, op):
    """The gradient against differences of the forward pass in fp32: along a random direction the derivative of
    L = sum(g . y) is (L(x + t d) - L(x - t d)) / 2t.  L is computed from results of fp32, each off by 32 units of its
    row's norm.  A unit vector along v + s d has a third derivative of at most 15 (|d| / |v|)^3, so the difference is off
    by at most 15 / 6 t^2 |g| |x| (|d| / |x|)^3 a row; rows of 64 normal values differ in length by less than 1.8."""
    g = torch.Generator().manual_seed(4)
    T, hq, hk, D = 9, 3, 2, 64
    pos = torch.randint(0, 1000, (T,), generator=g).cuda()
    inv = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()

    def rand(*shape):
        return torch.randn(*shape, generator=g).cuda()

    q, k, qw, kw = rand(T, hq, D), rand(T, hk, D), 1 + 0.2 * rand(D), 1 + 0.2 * rand(D)
    gq, gk = rand(T, hq, D), rand(T, hk, D)
    leaves = [v.requires_grad_(True) for v in ((q, k, qw, kw) if op == "norm" else (q, k))]

    def f(*v):
        if op == "norm":
            return torch.ops.b200ht.norm_rotary_qk(*v, pos, inv, 1e-6, None, "blocks", False, True)
        return torch.ops.b200ht.rotary_qk(*v, pos, inv, None, "blocks", False, True, False)

    def loss(*v):
        a, b = f(*v)
        return (a.double() * gq).sum() + (b.double() * gk).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    t = 2.0 ** -7
    scale = float(gq.double().norm() * q.detach().double().norm() + gk.double().norm() * k.detach().double().norm())
    with torch.no_grad():
        for i, (v, gv) in enumerate(zip(leaves, grads)):
            d = rand(*v.shape)
            up, down = ([x + t * d * s if j == i else x for j, x in enumerate(leaves)] for s in (1, -1))
            want = float((loss(*up) - loss(*down)) / (2 * t))
            got = float((gv.double() * d).sum())
            # 32 units of every row in both losses over 2t, and 15 / 6 * 1.8^3 < 16
            assert abs(got - want) <= scale * (64 * U / (2 * t) + 16 * t * t), (i, got, want)
    # only one result used: the other's gradient is missing
    a, _ = f(*leaves)
    only = torch.autograd.grad((a * gq).sum(), leaves, allow_unused=True)
    assert not only[1].any()


@pytest.mark.gpu
def test_registered_operators_check_and_compile(pkg):
    q, k, pos, inv = make(11, 4, 2, 64, 32, torch.bfloat16, packed=True, far=90)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.b200ht.rotary_qk, (q, k, pos, inv), test_utils=tests)
    torch.library.opcheck(torch.ops.b200ht.norm_rotary_qk, (q, k, w, w, pos, inv), test_utils=tests)
    torch._dynamo.reset()

    def f(q, k):
        a, b = torch.ops.b200ht.norm_rotary_qk(q, k, w, w, pos, inv, 1e-6, None, "blocks", False, True)
        return a * 2, b + 1

    for x, y in zip(torch.compile(f, fullgraph=True, backend="aot_eager")(q, k), f(q, k)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_graph_stream_and_repeat(pkg):
    """Captured and replayed twice side by side, on a stream of its own, and bit for bit the same on every call."""
    q, k, pos, inv = make(300, 8, 2, 128, 64, torch.bfloat16, packed=True, far=900)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def call():
        return (*pkg.norm_rotary_qk(q, k, w, w, pos, inv, hadamard=True),
                *pkg.norm_rotary_qk_backward(dq, dk, q, k, w, w, pos, inv, hadamard=True), *pkg.rotary_qk(q, k, pos, inv))

    want = call()
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


@pytest.mark.gpu
def test_results_lie_between_untouched_zones(pkg, lib):
    """Outputs inside larger buffers: nothing outside the rows is written."""
    l = lib.load()
    for T, hq, hk, D, pairs, dtype in ((3, 5, 2, 128, 64, torch.bfloat16), (9, 3, 1, 80, 40, torch.float32),
                                       (2, 1, 1, 66, 33, torch.float16), (65, 2, 2, 64, 16, torch.bfloat16)):
        q, k, pos, inv = make(T, hq, hk, D, pairs, dtype, packed=True, far=9)
        outs = [torch.full((T + 4, h + 1, D + 16), 7.0, dtype=dtype, device="cuda") for h in (hq, hk)]
        qo, ko = outs[0][2:2 + T, :hq, 8:8 + D], outs[1][2:2 + T, :hk, 8:8 + D]
        strides = (ctypes.c_longlong * 8)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), qo.stride(0), qo.stride(1),
                                          ko.stride(0), ko.stride(1))
        rc = l.b200ht_rotary_qk(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), None, None, 0.0, T, hq, hk, D, strides,
                                {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[dtype], pos.data_ptr(), 0, 1, 1, None,
                                inv.data_ptr(), pairs, lib.ROT_POS64, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.error_string(rc)
        assert_close(qo, forward64(q, None, 0, pos, inv))
        assert_close(ko, forward64(k, None, 0, pos, inv))
        for o, view in zip(outs, (qo, ko)):
            view.fill_(7.0)
            assert bool((o == 7.0).all())


@pytest.mark.gpu
def test_offsets_beyond_32_bits(pkg):
    """Rows 32768 elements apart: the last tokens lie behind element 2^31."""
    T, row = 65600, 32768
    big = torch.empty(T * row, dtype=torch.bfloat16, device="cuda")
    q, k = big.as_strided((T, 2, 128), (row, 128, 1)), big.as_strided((T, 1, 128), (row, 128, 1), 512)
    g = torch.Generator(device="cuda").manual_seed(5)
    q.copy_(torch.randn(T, 2, 128, generator=g, device="cuda"))
    k.copy_(torch.randn(T, 1, 128, generator=g, device="cuda"))
    pos, inv = torch.arange(T, device="cuda"), (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    last = slice(T - 70, T)
    want = [forward64(x[last], w, 1e-6, pos[last], inv, hadamard=True) for x in (q, k)]
    grads = pkg.norm_rotary_qk_backward(q, k, q, k, w, w, pos, inv)
    got = pkg.norm_rotary_qk(q, k, w, w, pos, inv, hadamard=True, inplace=True)
    for a, b in zip(got, want):
        assert_close(a[last], b)
    assert torch.isfinite(grads[0]).all() and grads[0].shape == q.shape
    # a kernel for other alignments walks the same offsets
    odd = big.as_strided((T, 1, 66), (row, 66, 1), 1001)
    odd.copy_(torch.randn(T, 1, 66, generator=g, device="cuda"))
    want = forward64(odd[last], None, 0, pos[last], inv[:33])
    assert_close(pkg.rotary_qk(odd, None, pos, inv[:33])[0][last], want)


@pytest.mark.gpu
def test_gradients_captured_in_a_graph(pkg):
    """A training step captured by torch.autograd.grad: forward, backward and replay with other values in the leaves."""
    q, k, pos, inv = make(40, 4, 2, 64, 32, torch.bfloat16, far=60)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, w, w)]

    def step():
        out = torch.ops.b200ht.norm_rotary_qk(*leaves, pos, inv, 1e-6, None, "blocks", False, True)
        return torch.autograd.grad(out, leaves, (dq, dk))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    torch.cuda.synchronize()
    with torch.no_grad():
        leaves[0].copy_(q.flip(0))
    with torch.cuda.stream(s):
        graph.replay()
    torch.cuda.synchronize()
    want = pkg.norm_rotary_qk_backward(dq, dk, q.flip(0), k, w, w, pos, inv, hadamard=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_backward_that_saved_what_was_overwritten_fails(pkg):
    """q and k are views of a projection that another operation has saved: its backward must not use the rotated values."""
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, k, pos, inv = make(7, 4, 2, 64, 32, torch.bfloat16, packed=True, far=50)
    scale = torch.ones(1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: pkg.rotary_qk(q, None, pos, inv, inplace=True), lambda: pkg.rotary_qk(k, q, pos, inv, inplace=True),
                 lambda: pkg.norm_rotary_qk(q, k, w, w, pos, inv, inplace=True)):
        y = (q._base * scale).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    y = (q._base * scale).sum()
    pkg.rotary_qk(q, k, pos, inv)
    y.backward()          # not in place: nothing was overwritten
    leaf = q.float().bfloat16().requires_grad_()
    with torch.no_grad():
        assert pkg.rotary_qk(leaf, None, pos, inv, inplace=True)[0] is leaf
    with torch.inference_mode():
        cache = q.clone()
        pkg.rotary_qk(cache, None, pos, inv, inplace=True)
    pkg.rotary_qk(cache, None, pos, inv, inplace=True)


@pytest.mark.gpu
def test_norm_without_keys(pkg):
    """None for the keys, or keys of no head, forward; keys of no head backward."""
    q, _, pos, inv = make(9, 4, 0, 64, 32, torch.bfloat16, far=40)
    w = torch.linspace(0.5, 1.5, 64, device="cuda").bfloat16()
    y, none = pkg.norm_rotary_qk(q, None, w, w, pos, inv, hadamard=True)
    assert none is None
    assert_close(y, forward64(q, w, 1e-6, pos, inv, hadamard=True))
    assert torch.equal(pkg.norm_rotary_qk(q, q[:, :0], w, w, pos, inv, hadamard=True)[0], y)
    with_keys = pkg.norm_rotary_qk_backward(q, q, q, q, w, w, pos, inv)
    without = pkg.norm_rotary_qk_backward(q, q[:, :0], q, q[:, :0], w, w, pos, inv)
    assert torch.equal(without[0], with_keys[0]) and without[1].shape == (9, 0, 64) and not without[3].any()


@pytest.mark.gpu
def test_frequencies_that_would_lose_their_gradient_are_refused(pkg):
    q, k, pos, inv = make(5, 4, 2, 64, 32, torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q.requires_grad_()
    for learn in (False, True):
        f = inv.clone().requires_grad_(learn)
        for y, _ in (torch.ops.b200ht.rotary_qk(q, k, pos, f), torch.ops.b200ht.norm_rotary_qk(q, k, w, w, pos, f)):
            if learn:
                with pytest.raises(RuntimeError, match="inv_freq has no gradient"):
                    y.float().sum().backward()
            else:
                q.grad = None
                y.float().sum().backward()
                assert q.grad.shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hk,D,pairs,dtype", [
    (4001, 8, 2, 128, 64, torch.bfloat16), (2500, 1, 64, 64, 32, torch.float16), (3000, 2, 1, 256, 128, torch.float32),
    (5000, 3, 3, 80, 40, torch.bfloat16), (3001, 64, 1, 66, 33, torch.bfloat16), (2000, 1, 1, 80, 20, torch.float32),
    (1, 1, 1, 128, 64, torch.bfloat16), (3, 0, 5, 96, 48, torch.float16),
])
def test_gradients_lie_between_untouched_zones(pkg, lib, T, hq, hk, D, pairs, dtype):
    """The gradients inside larger rows, the weights' and the workspace of just the size asked for with a pattern on both
    sides; enough tokens that the number of blocks, and so of the workspace's rows, reaches its limit."""
    l = lib.load()
    q, k, pos, inv = make(T, hq, hk, D, pairs, dtype, packed=True, far=99)
    w = torch.linspace(0.5, 1.5, D, device="cuda").to(dtype)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    outs = [torch.full((T + 4, h + 1, D + 16), 7.0, dtype=dtype, device="cuda") for h in (hq, hk)]
    dq, dk = outs[0][2:2 + T, :hq, 8:8 + D], outs[1][2:2 + T, :hk, 8:8 + D]
    need, guard = l.b200ht_norm_rotary_qk_backward_workspace_bytes(D), 4096
    ws = torch.full((need + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
    dw = torch.full((3, 2, D), 7.0, dtype=dtype, device="cuda")
    strides = (ctypes.c_longlong * 12)(*(s for x in (gq, gk, q, k, dq, dk) for s in x.stride()[:2]))
    rc = l.b200ht_norm_rotary_qk_backward(
        gq.data_ptr(), gk.data_ptr(), q.data_ptr(), k.data_ptr(), w.data_ptr(), w.data_ptr(), 1e-6, dq.data_ptr(), dk.data_ptr(),
        dw[1, 0].data_ptr(), dw[1, 1].data_ptr(), T, hq, hk, D, strides, {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[dtype],
        pos.data_ptr(), 0, 1, 1, None, inv.data_ptr(), pairs, lib.ROT_POS64, ws.data_ptr() + guard, need,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.error_string(rc)
    want = pkg.norm_rotary_qk_backward(gq, gk, q, k, w, w, pos, inv)
    for a, b in zip((dq, dk, dw[1, 0], dw[1, 1]), want):
        assert torch.equal(a, b)
    for z in (ws[:guard], ws[guard + need:]):
        assert bool((z == 0xA5).all())
    assert bool((dw[0] == 7.0).all() and (dw[2] == 7.0).all())
    for o, view in zip(outs, (dq, dk)):
        view.fill_(7.0)
        assert bool((o == 7.0).all())
