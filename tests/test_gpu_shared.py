"""fused_attention_decode_shared against softmax attention in 64 bits over the dequantised tiers.

Tolerances, derived. Every operand of a product is two truncated f16 parts: off by at most 2^-20 of it, and a product
leaves out lo lo, at most 2^-20 more: 3 (2^-20) in all, relative to the sum of the products' sizes. FP32 sums add a
half step (2^-24) per addition; a logit has at most 24 matrix instructions' results and their inner sums (256 channels,
3 products each) in its chain, so a logit is off by at most d_t = (3 (2^-20) + 56 (2^-24)) sum_c |q_c k_c| / sqrt(D)
plus its own rounding, |s_t| 2^-23. A weight is then off by 2 max d_t relative, an output by
(2 max d + 3 (2^-20) + chain) sum_t w_t |v_t|; the chain of a slot's accumulators and the merge of the slots have under 500
additions here: 2^-15. Weights: (2 max d + 2^-15) w."""
import ctypes

import pytest
import torch

from gpu_helpers import quantize_blocks_gpu

pytestmark = pytest.mark.gpu

KEYS = ("dense_K", "dense_V", "PBS_K_Packed", "PBS_K_Scales", "PBS_K_Zeroes", "PBS_V_Packed", "PBS_V_Scales",
        "PBS_V_Zeroes", "PBS_token_ids")


def make_tiers(g, nd, nb, hkv, d, kgs, fp16, mask="some", scale=1.0):
    """Tiers of nd FP32 tokens and nb blocks, and their keys, values and validity in 64 bits."""
    from tritiercache_amd import _C

    n = nb * kgs
    K = torch.randn((nd + n, hkv, d), generator=g, device="cuda") * scale
    K[:, :, :4] *= 4
    V = torch.randn((nd + n, hkv, d), generator=g, device="cuda") * scale
    t = {"dense_K": K[:nd].contiguous(), "dense_V": V[:nd].contiguous(), "dense_count": nd, "num_blocks": nb}
    valid = torch.ones(nd + n, dtype=torch.bool, device="cuda")
    if nb:
        packs = quantize_blocks_gpu(_C, K[nd:].contiguous(), V[nd:].contiguous(), kgs, fp16)
        ids = torch.arange(n, dtype=torch.int64, device="cuda")
        if mask == "some":
            ids[torch.rand(n, generator=g, device="cuda") < 0.2] = -1
            ids[-3:] = -1
        elif mask == "all":
            ids[:] = -1
        valid[nd:] = ids != -1
        t.update(zip(KEYS[2:], (*packs, ids)))
        meta = "fp16" if fp16 else "fp32"
        kk, vv = torch.empty((n, hkv, d), device="cuda"), torch.empty((n, hkv, d), device="cuda")
        _C.dequantize_k(*packs[:3], kk, nb, hkv, d, kgs, meta)
        _C.dequantize_v(*packs[3:], vv, n, hkv, d, meta)
        K, V = torch.cat([K[:nd], kk]), torch.cat([V[:nd], vv])
    return t, (K.double(), V.double(), valid)


def expected(q, parts, hkv):
    """(out, weights [Hq, tokens], sum w |v|, relative bound of the weights) over the tokens of `parts`."""
    hq, d = q.shape
    K = torch.cat([p[0] for p in parts]).transpose(0, 1)  # [Hkv, T, D]
    V = torch.cat([p[1] for p in parts]).transpose(0, 1)
    valid = torch.cat([p[2] for p in parts])
    x = q.double().view(hkv, hq // hkv, d)
    s = torch.where(valid, x @ K.transpose(1, 2) / d ** 0.5, -torch.inf)
    size = torch.where(valid, x.abs() @ K.abs().transpose(1, 2) / d ** 0.5, 0.0)
    if s.shape[-1] == 0 or not bool(valid.any()):
        z = torch.zeros((hq, d), dtype=torch.float64, device="cuda")
        return z, torch.zeros((hq, s.shape[-1]), dtype=torch.float64, device="cuda"), z, z[:, :1]
    w = torch.softmax(s, -1)
    off = (3 * 2.0 ** -20 + 56 * 2.0 ** -24) * size + 2.0 ** -23 * torch.where(valid, s.abs(), 0.0)
    rel = 2 * off.amax(-1) + 2.0 ** -15
    V = torch.where(valid[None, :, None], V, 0.0)
    return (w @ V).reshape(hq, d), w.reshape(hq, -1), (w @ V.abs()).reshape(hq, d), rel.reshape(hq, 1)


def check(got, mean, q, prefix, own, hkv, tag):
    out, w, size, rel = expected(q, [prefix, own], hkv)
    bound = (rel + 3 * 2.0 ** -20) * size + 2.0 ** -126
    off = (got.double() - out).abs()
    assert torch.isfinite(got).all(), tag
    assert bool((off <= bound).all()), (tag, float((off / bound).max()))
    if mean is not None:
        n = own[0].shape[0]
        ww = w[:, w.shape[1] - n:]
        off = (mean.double() - ww.mean(0)).abs()
        assert bool((off <= (ww * rel).mean(0) + 2.0 ** -126).all()), (tag, "weights")


def run(case, seed=1, mask="some", scale=1.0, weights=lambda i: i % 3 != 2, edit=None):
    """Builds the batch, runs it and checks every sequence. own: (FP32 tokens, blocks) of sequence i."""
    from tritiercache_amd import _C

    hq, hkv, d, b, (pd, pb), own, kgs, fp16 = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    prefix, pref = make_tiers(g, pd, pb, hkv, d, kgs, fp16, mask, scale)
    batch, refs = [], []
    for i in range(b):
        nd, nb = own(i)
        t, r = make_tiers(g, nd, nb, hkv, d, kgs, fp16, mask, scale)
        t["Q"] = torch.randn((hq, d), generator=g, device="cuda") * (1 + i % 3)
        t["attn_output"] = torch.full((hq, d), float("nan"), device="cuda")
        n = nd + nb * kgs
        t["mean_attn_weights"] = torch.full((n,), float("nan"), device="cuda") if n and weights(i) else None
        batch.append(t)
        refs.append(r)
    if edit:
        pref, refs = edit(prefix, pref, batch, refs)
    _C.fused_attention_decode_shared(prefix, batch, hq, hkv, d, kgs, "fp16" if fp16 else "fp32")
    torch.cuda.synchronize()
    for i, (t, r) in enumerate(zip(batch, refs)):
        check(t["attn_output"], t["mean_attn_weights"], t["Q"], pref, r, hkv, (case[:5], "sequence", i))
    return prefix, batch


def ragged(i):
    return (1 + 37 * i % 101, (0, 3, 1, 9)[i % 4])


CASES = [
    # Hq, Hkv, D, sequences, prefix (FP32 tokens, blocks), own, kgs, FP16 metadata
    (32, 8, 128, 1, (40, 10), ragged, 16, False),
    (32, 8, 128, 2, (264, 20), lambda i: (1, 0), 16, False),
    (32, 8, 128, 4, (300, 33), ragged, 16, True),     # one 16-row tile
    (32, 8, 128, 5, (300, 33), ragged, 32, True),     # 20 rows
    (32, 8, 128, 33, (31, 65), ragged, 16, False),    # 132 rows: two chunks
    (28, 4, 128, 64, (33, 100), ragged, 32, False),
    (16, 16, 128, 17, (1, 1), ragged, 16, True),      # one row per sequence and head
    (34, 2, 128, 3, (65, 7), ragged, 16, False),      # 17 heads per group
    (14, 2, 64, 23, (95, 51), ragged, 16, True),
    (9, 3, 64, 2, (0, 40), ragged, 32, False),
    (4, 4, 16, 3, (10, 5), ragged, 16, False),
    (4, 2, 48, 20, (33, 6), ragged, 32, True),
    (32, 32, 80, 17, (100, 30), ragged, 16, False),
    (12, 4, 96, 6, (257, 9), ragged, 16, True),
    (6, 2, 112, 40, (12, 31), ragged, 16, False),
    (4, 1, 144, 4, (64, 12), ragged, 16, False),
    (6, 3, 192, 50, (40, 20), ragged, 32, True),
    (4, 2, 208, 2, (31, 3), ragged, 16, True),
    (16, 8, 256, 12, (100, 40), ragged, 16, False),
    (16, 2, 256, 40, (5, 21), ragged, 16, True),
    (8, 2, 128, 65, (50, 12), ragged, 16, False),     # two launches
    (2, 1, 64, 130, (7, 3), lambda i: (i % 5, i % 2), 16, True),
    (32, 8, 128, 3, (0, 0), ragged, 16, False),       # no prefix
    (32, 8, 128, 3, (100, 9), lambda i: (0, 0), 16, False),  # nothing of their own
    (8, 2, 80, 20, (100, 0), lambda i: (0, i % 2), 16, True),
    (8, 8, 128, 6, (0, 1500), lambda i: (3, 200 * (i % 2)), 16, True),  # long
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c[:5] + c[6:]))
def test_against_64_bits(case):
    run(case)


# More sequences than a prefix is read one by one for: tiles of every kind, whole and short, alone and with others.
MANY = [(hq, hkv, d, b, (pd, pb), ragged, kgs, fp16)
        for (hq, hkv, d, b) in ((4, 2, 64, 33), (6, 1, 64, 64), (2, 2, 16, 40), (6, 2, 96, 40), (8, 1, 80, 50),
                                (3, 3, 128, 33), (6, 2, 128, 40), (7, 1, 128, 64), (2, 2, 144, 34), (9, 3, 256, 64))
        for (pd, pb, kgs, fp16) in ((1, 0, 16, False), (0, 1, 16, True), (31, 0, 16, True), (33, 3, 16, False),
                                    (64, 1, 32, True), (65, 35, 16, True), (0, 33, 32, False))]


@pytest.mark.parametrize("case", MANY, ids=lambda c: str(c[:5] + c[6:]))
def test_many_sequences_against_64_bits(case):
    run(case, seed=3, weights=lambda i: i % 16 == 1)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_many_sequences_masks_that_leave_nothing(d):
    own = lambda i: (0, i % 2)
    run((8, 2, d, 40, (20, 9), own, 16, False), mask="all")
    _, batch = run((8, 2, d, 40, (0, 9), own, 16, True), mask="all", weights=lambda i: True)
    for t in batch:
        assert bool((t["attn_output"] == 0).all())
        assert t["mean_attn_weights"] is None or bool((t["mean_attn_weights"] == 0).all())


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("fp16", [False, True])
def test_first_tiles_that_are_masked_or_tiny(d, fp16):
    """The scales of the prefix's parts come from its first tiles: these are masked, hold NaN there, or keys and values
    2^-20 (the FP32 ones' smallest 2^-100) of the later ones'."""
    def edit(prefix, pref, batch, refs):
        if not fp16:
            for x in (prefix["dense_K"], pref[0], prefix["dense_V"], pref[1]):
                x[:32] *= 2.0 ** -20
                x[3] *= 2.0 ** -80
        nd = prefix["dense_count"]
        prefix["PBS_token_ids"][:64] = -1
        pref[2][nd:nd + 64] = False
        prefix["PBS_K_Scales"][:4] = 0x7e00 if fp16 else float("nan")  # FP16 metadata: the bits of NaN, infinity
        prefix["PBS_V_Zeroes"][:64] = 0x7c00 if fp16 else float("inf")
        for x in pref[:2]:
            x[nd:nd + 64] = 0  # not attended
        return pref, refs

    run((8, 2, d, 40, (80, 40), ragged, 16, fp16), edit=edit)


@pytest.mark.parametrize("d,b", [(128, 3), (128, 30), (80, 9), (256, 20)])
def test_masks_that_leave_nothing(d, b):
    """Every packed slot masked: the FP32 tokens alone; without those, zeros (output and weights)."""
    run((8, 2, d, b, (20, 9), ragged, 16, False), mask="all")
    _, batch = run((8, 2, d, b, (0, 9), lambda i: (0, 3), 16, False), mask="all", weights=lambda i: True)
    for t in batch:
        assert bool((t["attn_output"] == 0).all()) and bool((t["mean_attn_weights"] == 0).all())
    _, batch = run((8, 2, d, b, (0, 0), lambda i: (0, 0), 16, False))
    assert all(bool((t["attn_output"] == 0).all()) for t in batch)


@pytest.mark.parametrize("b", [2, 25])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_masked_slots_may_hold_anything(d, b):
    """A block whose slots are all masked, with NaN and infinite scales and zeros, adds nothing."""
    def edit(prefix, pref, batch, refs):
        for t, r in [(prefix, pref)] + list(zip(batch, refs)):
            if not t["num_blocks"]:
                continue
            kgs = t["PBS_token_ids"].numel() // t["num_blocks"]
            nd = t["dense_count"]
            t["PBS_token_ids"][:kgs] = -1
            r[2][nd:nd + kgs] = False
            t["PBS_K_Scales"][0] = float("nan")
            t["PBS_K_Zeroes"][0] = float("inf")
            t["PBS_V_Scales"][:kgs] = float("inf")
            t["PBS_V_Zeroes"][:kgs] = float("nan")
            for x in r[:2]:
                x[nd:nd + kgs] = 0  # not attended
        return pref, refs

    run((8, 2, d, b, (33, 12), ragged, 16, False), edit=edit)


@pytest.mark.parametrize("b", [3, 40])
@pytest.mark.parametrize("scale", [1e-6, 1e5, 1e12])
def test_sizes_past_f16(scale, b):
    """Keys and values outside f16's range (queries scaled against them, so that the logits stay in reach)."""
    def edit(prefix, pref, batch, refs):
        for t in batch:
            t["Q"] /= scale
        return pref, refs

    run((8, 2, 128, b, (70, 12), ragged, 16, False), scale=scale, edit=edit)
    run((4, 4, 80, b, (70, 12), ragged, 16, False), scale=scale, edit=edit)


@pytest.mark.parametrize("b", [3, 40])
def test_one_large_token_among_small_ones(b):
    """A single large key and value inside a tile: the tiles around it keep their accuracy relative to sum w |v|."""
    def edit(prefix, pref, batch, refs):
        for x, r, f in ((prefix["dense_K"], pref[0], 3e4), (prefix["dense_V"], pref[1], 2e5)):
            x[50] *= f
            r[50] *= f
        for t in batch:
            t["Q"] *= 1e-3
        return pref, refs

    run((8, 2, 128, b, (90, 12), ragged, 16, False), edit=edit)


def test_the_shared_call_equals_calls_over_the_joined_tiers():
    """The same tokens as one cache per sequence, through the single-sequence call."""
    from tritiercache_amd import _C

    case = (32, 8, 128, 6, (200, 40), ragged, 16, False)
    hq, hkv, d, b, _, _, kgs, _ = case
    prefix, batch = run(case, seed=9)
    for t in batch:
        both = {}
        for k in KEYS:
            have = [x[k] for x in (prefix, t) if k in x]
            both[k] = torch.cat(have)
        out = torch.empty((hq, d), device="cuda")
        _C.fused_attention_decode(t["Q"], both["dense_K"], both["dense_V"], prefix["dense_count"] + t["dense_count"],
                                  *(both[k] for k in KEYS[2:]), prefix["num_blocks"] + t["num_blocks"], hq, hkv, d, out)
        torch.cuda.synchronize()
        assert float((out - t["attn_output"]).abs().max()) <= 2e-5 * float(out.abs().max())


def _call(prefix, batch, hq, hkv, d, kgs, fp16):
    """The C ABI call with tables of the caller's: (function of the stream, what must stay alive)."""
    from tritiercache_amd import _lib

    L = _lib.load()

    def fill(s, t):
        for k in KEYS:
            setattr(s, k, t[k].data_ptr() if k in t else None)
        s.dense_count, s.num_blocks = t["dense_count"], t["num_blocks"]

    p, seqs = _lib.DecodeSeq(), (_lib.DecodeSeq * len(batch))()
    fill(p, prefix)
    for s, t in zip(seqs, batch):
        fill(s, t)
        s.Q, s.attn_output = t["Q"].data_ptr(), t["attn_output"].data_ptr()
        s.mean_attn_weights = t["mean_attn_weights"].data_ptr() if t["mean_attn_weights"] is not None else None
    dev = torch.frombuffer(bytearray(bytes(seqs)), dtype=torch.uint8).cuda()
    size = L.tt_shared_decode_workspace_bytes(ctypes.byref(p), seqs, len(batch), hq, hkv, d, kgs)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN: nothing is read before it is written

    def go():
        s = torch.cuda.current_stream().cuda_stream
        _lib.check(L.tt_fused_attention_decode_shared(ctypes.byref(p), seqs, dev.data_ptr(), len(batch), hq, hkv, d, kgs,
                                                      int(fp16), ws.data_ptr(), size, s))
    return go, (p, seqs, dev, ws)


@pytest.mark.parametrize("case", [CASES[2], CASES[4], CASES[12], CASES[18], CASES[20]], ids=lambda c: str(c[:5]))
def test_replays_and_streams(case):
    """The C ABI call on another stream, and captured once and replayed on new data with eager work in between; each
    result equals the eager call's bit for bit (no atomics, a fixed order of sums)."""
    hq, hkv, d, b, _, _, kgs, fp16 = case
    prefix, batch = run(case, seed=4)
    go, keep = _call(prefix, batch, hq, hkv, d, kgs, fp16)

    def results():
        return [x.clone() for t in batch for x in (t["attn_output"], t["mean_attn_weights"]) if x is not None]

    want = results()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    g = torch.Generator(device="cuda").manual_seed(77)
    for i in range(4):
        for t in batch:
            t["Q"].copy_(torch.randn((hq, d), generator=g, device="cuda"))
            if t["dense_count"]:
                t["dense_V"].copy_(torch.randn(t["dense_V"].shape, generator=g, device="cuda"))
        go()
        torch.cuda.synchronize()
        want = results()
        for t in batch:
            t["attn_output"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results(), want)), i


@pytest.mark.parametrize("b", [2, 24])
def test_offsets_past_32_bits(b):
    """A packed prefix of more than 4 GiB of key words, all masked but its last blocks: the result is that of those
    blocks alone."""
    from tritiercache_amd import _C

    hq, hkv, d, kgs = 32, 32, 256, 16
    nb, tail = 131072 + 40, 24
    g = torch.Generator(device="cuda").manual_seed(6)
    small, ref = make_tiers(g, 0, tail, hkv, d, kgs, True, "none")
    big = {"dense_count": 0, "num_blocks": nb}
    for k in KEYS[2:]:
        per = small[k].shape[0] // tail
        x = torch.zeros((nb * per,) + tuple(small[k].shape[1:]), dtype=small[k].dtype, device="cuda")
        if k == "PBS_token_ids":
            x.fill_(-1)
        x[(nb - tail) * per:] = small[k]
        big[k] = x
    q = torch.randn((b, hq, d), generator=g, device="cuda")
    out = torch.empty((b, hq, d), device="cuda")
    batch = [{"Q": q[i], "attn_output": out[i], "dense_count": 0, "num_blocks": 0} for i in range(b)]
    _C.fused_attention_decode_shared(big, batch, hq, hkv, d, kgs, "fp16")
    torch.cuda.synchronize()
    none = tuple(x[:0] for x in ref)
    for i in range(b):
        check(out[i], None, q[i], ref, none, hkv, i)


def test_many_sequences_on_two_streams_with_a_workspace_each():
    case = (32, 8, 128, 33, (31, 65), ragged, 16, False)
    hq, hkv, d, _, _, _, kgs, fp16 = case
    prefix, batch = run(case, seed=12)
    want = [t["attn_output"].clone() for t in batch]
    other = [dict(t, attn_output=torch.zeros_like(t["attn_output"]),
                  mean_attn_weights=None if t["mean_attn_weights"] is None else torch.zeros_like(t["mean_attn_weights"]))
             for t in batch]
    calls = [_call(prefix, x, hq, hkv, d, kgs, fp16) for x in (batch, other)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for (go, _), s in zip(calls, streams):
            with torch.cuda.stream(s):
                go()
    torch.cuda.synchronize()
    for x in (batch, other):
        assert all(torch.equal(t["attn_output"], y) for t, y in zip(x, want))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b", [3, 40])
@pytest.mark.parametrize("fp16", [False, True])
def test_tiers_at_any_element(d, b, fp16):
    """Tiers that begin at the second element of their memory: no alignment but the element's."""
    def moved(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        y.copy_(x)
        return y

    def edit(prefix, pref, batch, refs):
        for t in [prefix, *batch]:
            for k in KEYS + ("Q", "attn_output", "mean_attn_weights"):
                if isinstance(t.get(k), torch.Tensor) and t[k].numel():
                    t[k] = moved(t[k])
        return pref, refs

    run((8, 2, d, b, (70, 13), ragged, 16, fp16), seed=8, edit=edit)


@pytest.mark.parametrize("b", [2, 40])
def test_a_long_fp32_prefix(b):
    """FP32 tiers of more than 4 GiB: zeros (logits 0, values 0) but for the last tokens, so that a sequence's output is
    sum e^s v / (zeros + sum e^s) over those."""
    from tritiercache_amd import _C

    hq, hkv, d, nd, tail = 32, 32, 256, 131072 + 333, 37
    g = torch.Generator(device="cuda").manual_seed(16)
    K, V = (torch.zeros((nd, hkv, d), device="cuda") for _ in range(2))
    K[-tail:] = torch.randn((tail, hkv, d), generator=g, device="cuda")
    V[-tail:] = torch.randn((tail, hkv, d), generator=g, device="cuda")
    q = torch.randn((b, hq, d), generator=g, device="cuda") * 3
    out = torch.empty((b, hq, d), device="cuda")
    batch = [{"Q": q[i], "attn_output": out[i], "dense_count": 0, "num_blocks": 0} for i in range(b)]
    _C.fused_attention_decode_shared({"dense_K": K, "dense_V": V, "dense_count": nd, "num_blocks": 0}, batch, hq, hkv, d)
    torch.cuda.synchronize()
    k, v = K[-tail:].double().transpose(0, 1), V[-tail:].double().transpose(0, 1)  # [heads, tail, D]
    for i in range(b):
        x = q[i].double()[:, None]
        s = (x @ k.transpose(1, 2))[:, 0] / d ** 0.5
        size = (x.abs() @ k.abs().transpose(1, 2))[:, 0] / d ** 0.5
        w = torch.exp(s) / (nd - tail + torch.exp(s).sum(-1, keepdim=True))
        off = (3 * 2.0 ** -20 + 56 * 2.0 ** -24) * size + 2.0 ** -23 * s.abs()
        rel = 2 * off.amax(-1, keepdim=True) + 2.0 ** -15  # as in expected()
        want, mag = (w[:, None] @ v)[:, 0], (w[:, None] @ v.abs())[:, 0]
        assert bool(((out[i].double() - want).abs() <= (rel + 3 * 2.0 ** -20) * mag + 2.0 ** -126).all()), i


def test_more_rows_than_a_workgroup_takes():
    """128 query heads of one KV head, 64 sequences: 8192 rows."""
    run((128, 1, 64, 64, (70, 21), lambda i: (1 + i % 3, i % 2), 16, False), seed=9, weights=lambda i: i == 5)


# Few rows behind long prefixes: a wave's tiles are its own. Tiles that start and end anywhere, both kinds, masked ones.
LONG = [(8, 8, 128, 3, (1000, 3001), ragged, 16, True), (32, 8, 64, 8, (33, 1100), ragged, 32, False),
        (32, 32, 80, 5, (700, 250), lambda i: (i, i % 2), 16, True), (12, 12, 96, 32, (1, 600), lambda i: (i % 7, 0), 16, False),
        (32, 32, 16, 9, (5, 501), lambda i: (i, 0), 16, True), (28, 4, 128, 4, (0, 3500), ragged, 16, False),
        (16, 16, 112, 2, (2500, 400), lambda i: (0, i), 32, True), (4, 1, 128, 8, (12000, 0), ragged, 16, False)]


@pytest.mark.parametrize("case", LONG, ids=lambda c: str(c[:5] + c[6:]))
def test_few_rows_behind_a_long_prefix(case):
    run(case, seed=21, weights=lambda i: i % 4 == 1)


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("fp16", [False, True])
def test_few_rows_masked_first_tiles_and_sizes(d, fp16):
    """Masked first tiles with NaN scales, then tiles a thousand times larger than those before them."""
    def edit(prefix, pref, batch, refs):
        nd = prefix["dense_count"]
        prefix["PBS_token_ids"][:64] = -1
        pref[2][nd:nd + 64] = False
        prefix["PBS_K_Scales"][:4] = 0x7e00 if fp16 else float("nan")
        prefix["PBS_V_Zeroes"][:64] = 0x7c00 if fp16 else float("inf")
        for x in pref[:2]:
            x[nd:nd + 64] = 0  # not attended
        for x, r in ((prefix["dense_K"], pref[0]), (prefix["dense_V"], pref[1])):
            for at, f in ((100, 1e3), (101, 1e6), (150, 1e9)):
                x[at:] *= f
                r[at:nd] *= f
        for t in batch:
            t["Q"] *= 1e-18
        return pref, refs

    run((8, 8, d, 6, (200, 3000), ragged, 16, fp16), seed=22, edit=edit, weights=lambda i: i % 4 == 1)
