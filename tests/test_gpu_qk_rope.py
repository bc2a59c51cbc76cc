"""qk_norm_rope against its formula in 64 bits: every type, odd and partial rotations, strides, scattered rows,
positions outside the tables, in place, streams and replayed graphs.

Tolerances, derived. An output is FP32 arithmetic rounded once to its type, at most half a step: eps / 2 of the value.
The FP32 part: an input, weight or table value enters exactly. y = x r w has the roundings of the mean of squares (a
sum of D <= 256 products in chains of at most 16 fused adds and 4 more, all terms positive: at most 20 half steps, half of
that behind the root), the division, the sum with eps, the root (one step) and two products: under 16 half steps of FP32,
relative. z = y c - y' s: two products' errors and the sum's, relative to |y c| + |y' s|. So
|got - exact| <= (eps_out / 2) |exact| + 20 (2^-24) (|y c| + |y' s|) plus half the smallest step of the output's type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def tables(rows, rot, dtype, g):
    a = torch.rand((rows, rot), generator=g, device="cuda", dtype=torch.float64) * 6.3
    return a.cos().to(dtype), a.sin().to(dtype)  # halves of their own: both are read


def formula(x, w, cos, sin, eps):
    """(z, |y c| + |y' s|) in 64 bits; cos, sin [tokens, rot] or None."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    z, mag = x.clone(), x.abs()
    if cos is not None:
        rot = cos.shape[1]
        h = rot // 2
        c, s = cos.double()[:, None], sin.double()[:, None]
        a, b = x[..., :h], x[..., h:rot]
        z[..., :h], mag[..., :h] = a * c[..., :h] - b * s[..., :h], (a * c[..., :h]).abs() + (b * s[..., :h]).abs()
        z[..., h:rot] = b * c[..., h:] + a * s[..., h:]
        mag[..., h:rot] = (b * c[..., h:]).abs() + (a * s[..., h:]).abs()
    return z, mag


def check(got, z, mag, tag):
    t = got.dtype
    bound = torch.finfo(t).eps / 2 * z.abs() + 20 * 2.0 ** -24 * mag + TINY[t] / 2
    off = (got.double() - z).abs()
    assert torch.isfinite(got).all(), tag
    assert bool((off <= bound).all()), (tag, float((off / bound.clamp_min(1e-300)).max()))


def inputs(seed, tokens, hq, hkv, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = lambda h: (torch.randn((tokens, h, d), generator=g, device="cuda") * 3).to(dtype)  # noqa: E731
    return g, x(hq), x(hkv), x(hkv)


# tokens, hq, hkv, d, rot, norms, in, out, table, weight
CASES = [
    (1, 32, 8, 128, 128, True, BF16, F32, F32, BF16),
    (1, 1, 1, 16, 16, True, F32, F32, F32, F32),
    (3, 5, 1, 16, 0, True, F16, F16, F32, F32),
    (7, 4, 2, 32, 16, False, F32, BF16, BF16, F32),
    (65, 14, 2, 64, 64, True, BF16, BF16, BF16, BF16),
    (33, 3, 3, 48, 48, True, F16, F32, F16, F16),
    (130, 32, 32, 80, 32, False, F32, F32, F32, F32),
    (17, 12, 4, 96, 96, True, F32, F16, F16, BF16),
    (9, 7, 7, 112, 80, True, BF16, F16, F32, F32),
    (1000, 28, 4, 128, 64, False, F16, BF16, BF16, F32),
    (5, 6, 2, 144, 144, True, F32, F32, BF16, F32),
    (21, 4, 2, 208, 48, True, F16, F32, F32, F16),
    (300, 16, 8, 256, 256, True, BF16, F32, BF16, BF16),
    (4099, 9, 3, 64, 64, True, F32, F32, F32, F32),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_formula(case):
    from tritiercache_amd import _C

    tokens, hq, hkv, d, rot, norms, src, dst, tab, wt = case
    g, q, k, v = inputs(11, tokens, hq, hkv, d, src)
    cos, sin = tables(tokens, rot, tab, g) if rot else (None, None)
    qw, kw = ((torch.randn((2, d), generator=g, device="cuda")).to(wt).unbind(0)) if norms else (None, None)
    qo, ko, vo = _C.qk_norm_rope(q, k, v, cos, sin, q_weight=qw, k_weight=kw, eps=1e-5, out_dtype=dst)
    check(qo, *formula(q, qw, cos, sin, 1e-5), ("q", case))
    check(ko, *formula(k, kw, cos, sin, 1e-5), ("k", case))
    assert torch.equal(vo, v.to(dst))


@pytest.mark.parametrize("hq,hkv,d,rot,src,dst", [(5, 3, 128, 128, BF16, BF16), (9, 2, 256, 64, F16, BF16),
                                                  (14, 2, 80, 80, F16, F16), (1, 1, 16, 0, BF16, F16)], ids=str)
def test_many_tokens_of_16_bits(hq, hkv, d, rot, src, dst):
    """Views of a joint projection at odd elements, keys and values scattered, as many tokens as several heads of one
    share a lane group for."""
    from tritiercache_amd import _C

    tokens = 140000 if d == 16 else 9001
    g = torch.Generator(device="cuda").manual_seed(d)
    joint = torch.randn(tokens * (hq + 2 * hkv) * d + 1, generator=g, device="cuda").to(src)[1:]
    joint = joint.view(tokens, hq + 2 * hkv, d)
    q, k, v = joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]
    cos, sin = tables(500, rot, F32, g) if rot else (None, None)
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda")
    qw, kw = torch.randn((2, d), generator=g, device="cuda").to(BF16).unbind(0)
    rows = torch.randperm(tokens + 5, generator=g, device="cuda")[:tokens]
    rows[::7] = -1
    tier_k, tier_v = (torch.full((tokens + 5, hkv, d), 7.0, dtype=dst, device="cuda") for _ in range(2))
    qo, _, _ = _C.qk_norm_rope(q, k, v, cos, sin, pos, qw, kw, rows=rows, k_out=tier_k, v_out=tier_v)
    at = (cos[pos], sin[pos]) if rot else (None, None)
    check(qo, *formula(q, qw, *at, 1e-6), "q")
    z, mag = formula(k, kw, *at, 1e-6)
    stored = rows >= 0
    check(tier_k[rows[stored]], z[stored], mag[stored], "k")
    assert torch.equal(tier_v[rows[stored]], v[stored].to(dst))
    free = torch.ones(tokens + 5, dtype=torch.bool, device="cuda")
    free[rows[stored]] = False
    assert bool((tier_k[free] == 7).all()) and bool((tier_v[free] == 7).all())
    if src == dst:
        want = qo.clone()
        _C.qk_norm_rope(q, k, None, cos, sin, pos, qw, kw, q_out=q, k_out=torch.empty_like(k))
        assert torch.equal(q, want)


@pytest.mark.parametrize("dst", [F32, BF16], ids=str)
def test_views_positions_and_rows(dst):
    """Views of a joint projection, positions of the sequences' own, rows of a tier: padded tokens and rows outside it
    leave the tier as it was, positions outside the tables give NaN."""
    from tritiercache_amd import _C

    tokens, hq, hkv, d, rot, room = 40, 8, 2, 128, 96, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    # the rows start at odd elements: no 16-byte alignment
    joint = torch.randn(tokens * (hq + 2 * hkv) * d + 1, generator=g, device="cuda").to(F16)[1:]
    joint = joint.view(tokens, hq + 2 * hkv, d)
    q, k, v = joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]
    cos, sin = tables(200, rot, F32, g)
    pos = torch.randint(0, 200, (tokens,), generator=g, device="cuda")
    pos[7], pos[9], pos[11] = 200, -1, 2 ** 40
    rows = torch.randperm(room, generator=g, device="cuda")[:tokens]
    rows[0], rows[3], rows[5] = -1, room, -2 ** 40
    kw = torch.rand(d, generator=g, device="cuda") + 0.5
    tier_k, tier_v = (torch.full((room, hkv, d + 3), 7.0, dtype=dst, device="cuda")[..., :d] for _ in range(2))
    qo, ko, vo = _C.qk_norm_rope(q, k, v, cos, sin, pos, None, kw, rows=rows, out_dtype=dst, k_out=tier_k, v_out=tier_v)
    assert ko is tier_k and vo is tier_v
    lost = [7, 9, 11]
    keep = torch.tensor([t not in lost for t in range(tokens)], device="cuda")
    at = pos.clamp(0, 199)
    zq, mq = formula(q, None, cos[at], sin[at], 1e-6)
    zk, mk = formula(k, kw, cos[at], sin[at], 1e-6)
    check(qo[keep], zq[keep], mq[keep], "q")
    assert torch.isnan(qo[lost]).all()
    stored = (rows >= 0) & (rows < room)
    check(ko[rows[stored & keep]], zk[stored & keep], mk[stored & keep], "k")
    gone = [t for t in lost if bool(stored[t])]
    assert torch.isnan(ko[rows[gone]]).all()
    assert torch.equal(vo[rows[stored]], v[stored].to(dst))
    free = torch.ones(room, dtype=torch.bool, device="cuda")
    free[rows[stored]] = False
    assert bool((ko[free] == 7).all()) and bool((vo[free] == 7).all())
    assert bool((tier_k.as_strided((room, hkv, 3), (hkv * (d + 3), d + 3, 1), d) == 7).all())


def test_transposed_outputs_in_place_and_no_values():
    from tritiercache_amd import _C

    g, q, k, _ = inputs(5, 70, 6, 3, 64, BF16)
    cos, sin = tables(70, 64, BF16, g)
    zq, zk = formula(q, None, cos, sin, 0), formula(k, None, cos, sin, 0)
    qt = torch.empty((6, 70, 64), dtype=BF16, device="cuda").transpose(0, 1)
    kt = torch.empty((3, 70, 64), dtype=BF16, device="cuda").transpose(0, 1)
    qo, ko, vo = _C.qk_norm_rope(q, k, None, cos, sin, q_out=qt, k_out=kt)
    assert vo is None
    check(qo, *zq, "q")
    check(ko, *zk, "k")
    q2, k2 = q.clone(), k.clone()
    _C.qk_norm_rope(q2, k2, None, cos, sin, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


def test_zeros_large_and_non_finite_rows():
    """A row of zeros stays zero under the norm; squares that pass FP32 give what the formula in FP32 gives (zeros);
    NaN and infinities stay in their rows."""
    from tritiercache_amd import _C

    g, q, k, v = inputs(6, 8, 4, 4, 128, F32)
    w = torch.ones(128, device="cuda")
    cos, sin = tables(8, 128, F32, g)
    q[0, 0] = 0
    q[1, 1] = 1e25
    q[2, 2, 5] = float("nan")
    q[3, 3, 70] = float("inf")
    qo, _, _ = _C.qk_norm_rope(q, k, v, cos, sin, q_weight=w, k_weight=w)
    assert bool((qo[0, 0] == 0).all()) and bool((qo[1, 1] == 0).all())
    assert torch.isnan(qo[2, 2]).all()
    others = [c for c in range(128) if c not in (6, 70)]  # the infinity's pair
    assert torch.isnan(qo[3, 3, 70]) and bool((qo[3, 3, others] == 0).all())
    fine = torch.ones((8, 4), dtype=torch.bool, device="cuda")
    fine[1, 1] = fine[2, 2] = fine[3, 3] = False
    z, mag = formula(q, w, cos, sin, 1e-6)
    check(qo[fine], z[fine], mag[fine], "the other rows")


def test_no_tokens():
    from tritiercache_amd import _C

    q, k = torch.empty((0, 4, 64), device="cuda"), torch.empty((0, 2, 64), device="cuda")
    qo, ko, vo = _C.qk_norm_rope(q, k, k.clone())
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64) and vo.shape == (0, 2, 64)


def test_streams_and_replays():
    """On the current stream, and captured once and replayed on new data with eager work in between."""
    from tritiercache_amd import _C

    g, q, k, v = inputs(8, 50, 8, 2, 128, BF16)
    cos, sin = tables(50, 128, F32, g)
    w = torch.rand(128, generator=g, device="cuda")
    want = _C.qk_norm_rope(q, k, v, cos, sin, q_weight=w, k_weight=w, out_dtype=F32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _C.qk_norm_rope(q, k, v, cos, sin, q_weight=w, k_weight=w, out_dtype=F32)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = [torch.zeros_like(x) for x in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _C.qk_norm_rope(q, k, v, cos, sin, q_weight=w, k_weight=w, q_out=outs[0], k_out=outs[1], v_out=outs[2])
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        want = _C.qk_norm_rope(q, k, v, cos, sin, q_weight=w, k_weight=w, out_dtype=F32)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_offsets_past_32_bits():
    """A tier whose last rows lie more than 2^32 bytes (and 2^31 elements) from its first."""
    from tritiercache_amd import _C

    d, hkv = 256, 8
    room = (1 << 31) // (hkv * d) + 11
    tier = torch.empty((room, hkv, d), dtype=BF16, device="cuda")
    tier[-3:] = 5
    tier[:2] = 5
    g, q, k, v = inputs(9, 2, 8, hkv, d, F32)
    rows = torch.tensor([room - 2, 0], device="cuda")
    _C.qk_norm_rope(q, k, v, rows=rows, q_out=torch.empty_like(q, dtype=BF16), k_out=tier, v_out=torch.empty_like(tier))
    assert torch.equal(tier[room - 2], k[0].to(BF16)) and torch.equal(tier[0], k[1].to(BF16))
    assert bool((tier[room - 3] == 5).all()) and bool((tier[room - 1] == 5).all()) and bool((tier[1] == 5).all())
