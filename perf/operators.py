"""Operators of a decode step for sequences that share a prompt, and the work their speed is measured on.

rope: norms of queries and keys for each head, the position rotation and the cast, with the keys and values written
to their rows of an FP32 tier (tt_qk_norm_rope). shared: decode attention of a batch over the tiers of a common
prefix and each sequence's own tiers (tt_fused_attention_decode_shared). Where `own` is false both are computed in
elementary torch operations in 32 bits. Inputs are synthetic and made on the GPU from a seed: N(0, 1) values, four key
channels of each KV head scaled by 8 (the outliers that 2-bit caches meet).
"""
import ctypes
import math
import random

import torch

own = False

SINK, RECENT, HEAVY = 4, 256, 0.05  # the HF patch's sinks, recent window and heavy-hitter share
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}  # the C ABI's type numbers


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _rope(hq, hkv, d, tokens, rot, norm, src, dst, table, fused, slots):
    """`fused`: q, k and v are views of one projection's output. `slots`: keys and values go to rows of a tier with
    room for more tokens, some tokens of the batch are padding and have none, positions are the sequences' own."""
    return {"kind": "rope", "hq": hq, "hkv": hkv, "d": d, "tokens": tokens, "rot": rot, "norm": norm, "src": src,
            "dst": dst, "table": table, "fused": fused, "slots": slots}


def _shared(hq, hkv, d, seqs, prefix, dense, blocks, lengths, kgs, meta, weights):
    """`prefix`: tokens of the prompt, split into tiers as an engine holds them. `dense`, `blocks`: the most FP32
    tokens and packed blocks of a sequence's own; each has between a quarter and all of them."""
    return {"kind": "shared", "hq": hq, "hkv": hkv, "d": d, "seqs": seqs, "prefix": prefix, "dense": dense,
            "blocks": blocks, "lengths": lengths, "kgs": kgs, "meta": meta, "weights": weights}


def listed():
    return [
        # One decode token of one sequence with 32/8 heads, bfloat16 projections, float32 vectors for the engine:
        # launch latency.
        {"name": "rope-1", **_rope(32, 8, 128, 1, 128, True, "bf16", "f32", "f32", False, False)},
        # A decode step of 61 sequences, views of one projection, keys and values appended to the sequences' tiers.
        {"name": "rope-61-append", **_rope(28, 4, 128, 61, 128, False, "f16", "f32", "f32", True, True)},
        # An odd prompt at head_dim 80 with 32 rotated channels, float32 throughout, no norms.
        {"name": "rope-1777-hd80", **_rope(32, 32, 80, 1777, 32, False, "f32", "f32", "f32", False, False)},
        # A prompt of 32k tokens with norms, bfloat16 in and out (what the prompt's own attention takes).
        {"name": "rope-32k", **_rope(32, 8, 128, 32768, 128, True, "bf16", "bf16", "bf16", True, False)},
        # Two sequences that begin to differ behind a short prompt: latency.
        {"name": "shared-2x580", **_shared(32, 8, 128, 2, 580, 1, 0, 1, 16, "fp32", True)},
        # Eight continuations of an 8k document, FP16 metadata (the engine's default).
        {"name": "shared-8x8k", **_shared(32, 8, 128, 8, 8192, 300, 20, 2, 16, "fp16", True)},
        # A serving batch behind a 32k system prompt, FP32 metadata, a few hundred own tokens each.
        {"name": "shared-64x32k", **_shared(32, 8, 128, 64, 32768, 280, 16, 3, 16, "fp32", True)},
        # The same prompt length with head_dim 64, 14/2 heads, blocks of 32 and a batch that fills no tile.
        {"name": "shared-23x32k-hd64", **_shared(14, 2, 64, 23, 32700, 270, 9, 4, 32, "fp16", True)},
        # head_dim 256 with two query heads per KV head at 8k.
        {"name": "shared-12x8k-hd256", **_shared(16, 8, 256, 12, 8192, 260, 4, 5, 16, "fp32", False)},
        # Multi-head attention with head_dim 80 at 2k.
        {"name": "shared-17x2k-hd80", **_shared(32, 32, 80, 17, 2048, 100, 3, 6, 16, "fp32", True)},
        # Long context: 32 questions about one 128k text, 28/4 heads.
        {"name": "shared-32x128k", **_shared(28, 4, 128, 32, 131072, 300, 8, 7, 16, "fp32", False)},
    ]


# (query heads, KV heads, head_dim) of the repository's benchmark configurations and tests
_HEADS = ((32, 8, 128), (32, 32, 128), (28, 4, 128), (40, 10, 128), (16, 8, 128), (32, 8, 64), (14, 2, 64),
          (9, 3, 64), (16, 8, 256), (8, 4, 256), (32, 32, 80), (32, 32, 96), (12, 4, 96))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    hq, hkv, d = rng.choice(_HEADS)
    if rng.random() < 0.35:
        src, dst = rng.choice((("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("f32", "f32")))
        most = 32768 * 48 * 128 * 4 // ((hq + 2 * hkv) * d * (_size(src) + _size(dst)))
        tokens = _log_int(rng, 1, min(most, 32768))
        rot = rng.choice((d, d, 16 * rng.randint(1, d // 16)))
        return _rope(hq, hkv, d, tokens, rot, rng.random() < 0.5, src, dst, rng.choice(("f32", src)),
                     rng.random() < 0.5, rng.random() < 0.5)
    seqs = _log_int(rng, 2, 64)
    prefix = _log_int(rng, 300, min(131072, 32 * 131072 * 28 * 128 // (seqs * hq * d), 131072 * 4 * 128 // (hkv * d)))
    kgs = rng.choice((16, 16, 32))
    return _shared(hq, hkv, d, seqs, prefix, _log_int(rng, 1, 300), rng.randint(0, 20), rng.randint(1, 1 << 20), kgs,
                   rng.choice(("fp32", "fp16")), rng.random() < 0.7)


def _size(name):
    return 4 if name == "f32" else 2


def _tiers(case):
    """FP32 tokens, packed blocks and masked slots of the prefix: sinks, recent window and heavy hitters in FP32, the
    rest packed, the last block filled up with masked slots."""
    n, kgs = case["prefix"], case["kgs"]
    dense = min(n, SINK + RECENT + math.ceil(HEAVY * n))
    blocks = -(-(n - dense) // kgs)
    return dense, blocks, blocks * kgs - (n - dense)


def _lengths(case):
    """FP32 tokens (the new one among them) and packed blocks of each sequence's own."""
    r = random.Random(case["lengths"])
    return [(r.randint(-(-case["dense"] // 4), case["dense"]), r.randint(case["blocks"] // 4, case["blocks"]))
            for _ in range(case["seqs"])]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rope":
        n = case["tokens"] * (hq + 2 * hkv) * d
        tables = 2 * case["tokens"] * case["rot"] * _size(case["table"])
        return {"bytes": n * (_size(case["src"]) + _size(case["dst"])) + tables + (16 * case["tokens"] if case["slots"] else 0),
                "flops": 10 * n}
    kgs, m = case["kgs"], 2 if case["meta"] == "fp16" else 4
    pd, pb, _ = _tiers(case)
    rows = [(pd, pb)] + _lengths(case)
    dense, blocks = sum(x for x, _ in rows), sum(x for _, x in rows)
    packed = blocks * (kgs * hkv * d // 2 + 2 * m * hkv * d + 2 * m * kgs * hkv + 8 * kgs)
    attended = case["seqs"] * (pd + pb * kgs) + sum(x + y * kgs for x, y in rows[1:])
    return {"bytes": 8 * dense * hkv * d + packed + 8 * case["seqs"] * hq * d
            + (4 * sum(x + y * kgs for x, y in rows[1:]) if case["weights"] else 0),
            "flops": 4 * hq * d * attended}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_rope(case, g):
    hq, hkv, d, n, rot = (case[k] for k in ("hq", "hkv", "d", "tokens", "rot"))
    src, dst = DTYPES[case["src"]], DTYPES[case["dst"]]
    make = lambda h: torch.randn((n, h, d), generator=g, device="cuda").to(src)  # noqa: E731
    s = {"case": case}
    if case["fused"]:
        qkv = make(hq + 2 * hkv)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        s["q"], s["k"], s["v"] = make(hq), make(hkv), make(hkv)
    if case["norm"]:
        s["qw"], s["kw"] = (1 + 0.2 * torch.randn((2, d), generator=g, device="cuda")).to(src).unbind(0)
    # a table of the rotation as models keep it: angles in 64 bits, both halves alike
    rows = max(n, 4096)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.cat([angle, angle], 1)
    s["cos"], s["sin"] = angle.cos().to(DTYPES[case["table"]]), angle.sin().to(DTYPES[case["table"]])
    s["out_rows"] = n
    if case["slots"]:
        s["out_rows"] = n + n // 2 + 1
        s["rows"] = torch.randperm(s["out_rows"], generator=g, device="cuda")[:n]
        s["rows"][torch.rand(n, generator=g, device="cuda") < 0.1] = -1
        s["positions"] = torch.randint(0, rows, (n,), generator=g, device="cuda")
    s["q_out"] = torch.zeros((n, hq, d), dtype=dst, device="cuda")
    # one row more than the tier has: where the plain form puts the tokens without a row
    s["k_out"], s["v_out"] = (torch.zeros((s["out_rows"] + 1, hkv, d), dtype=dst, device="cuda") for _ in range(2))
    if own:
        s["call"] = _rope_call(s)
    return s


def _words(codes, dim):
    """16 codes along `dim` to one int32 each, code i at bits 2 i."""
    shift = (2 * torch.arange(16, device=codes.device, dtype=torch.int32)).view(
        [16 if i == dim else 1 for i in range(codes.dim())])
    return (codes.to(torch.int32) << shift).sum(dim, dtype=torch.int32)


def _scales(lo, hi, meta):
    s = ((hi - lo) / torch.full_like(hi, 3.0)).clamp_min(1e-9)
    if meta == "fp16":
        return s, s.to(torch.float16).view(torch.uint16), lo.to(torch.float16).view(torch.uint16)
    return s, s, lo


def _keys(g, n, h, d):
    k = torch.randn((n, h, d), generator=g, device="cuda")
    for j in range(h):
        k[:, j, torch.randperm(d, generator=g, device="cuda")[:4]] *= 8.0
    return k


def _values(g, n, h, d):
    return torch.randn((n, h, d), generator=g, device="cuda")


def _packed(g, case, blocks):
    """Packed blocks of N(0, 1) keys and values in the layout of the quantisers."""
    h, d, kgs, meta = case["hkv"], case["d"], case["kgs"], case["meta"]
    n = blocks * kgs
    x = _keys(g, n, h, d).view(-1, kgs, h, d)
    lo = x.amin(1) if n else x.new_zeros((0, h, d))
    s, ks, kz = _scales(lo, x.amax(1) if n else lo, meta)
    kp = _words(torch.round((x - lo[:, None]) / s[:, None]).clamp_(0, 3).view(-1, kgs // 16, 16, h, d), 2)
    v = _values(g, n, h, d)
    lo = v.amin(2)
    s, vs, vz = _scales(lo, v.amax(2), meta)
    vp = _words(torch.round((v - lo[..., None]) / s[..., None]).clamp_(0, 3).view(n, h, d // 16, 16), 3)
    return {"kp": kp, "ks": ks, "kz": kz, "vp": vp, "vs": vs, "vz": vz}


def _prepare_shared(case, g):
    hq, hkv, d, kgs, b = (case[k] for k in ("hq", "hkv", "d", "kgs", "seqs"))
    pd, pb, masked = _tiers(case)
    s = {"case": case, "pd": pd, "pb": pb, "lengths": _lengths(case)}
    s["prefix"] = {"dk": _keys(g, pd, hkv, d), "dv": _values(g, pd, hkv, d), **_packed(g, case, pb)}
    s["prefix"]["ids"] = torch.arange(pd, pd + pb * kgs, dtype=torch.int64, device="cuda")
    if masked:
        s["prefix"]["ids"][-masked:] = -1
    # the sequences' own tiers: a slab each, so many rows of it in use
    cd, cb = case["dense"], case["blocks"]
    s["own"] = {"dk": _keys(g, b * cd, hkv, d), "dv": _values(g, b * cd, hkv, d), **_packed(g, case, b * cb)}
    ids = torch.arange(b * cb * kgs, dtype=torch.int64, device="cuda").view(b, cb * kgs)
    ids[torch.rand((b, cb * kgs), generator=g, device="cuda") < 0.05] = -1  # promoted to heavy hitters since
    s["own"]["ids"] = ids
    s["q"] = torch.randn((b, hq, d), generator=g, device="cuda")
    s["out"] = torch.zeros((b, hq, d), device="cuda")
    nd, nb = (torch.tensor(x, device="cuda")[:, None] for x in zip(*s["lengths"]))
    wide = cd + cb * kgs
    col = torch.arange(wide, device="cuda")[None]
    s["live"] = torch.cat([col[:, :cd] < nd, (col[:, :cb * kgs] < nb * kgs) & (ids != -1)], 1)
    # a sequence's weights are its FP32 tokens' and, right behind them, its packed slots'
    s["column"] = torch.where(col < nd, col, (col - nd + cd).clamp_max(wide - 1))
    s["used"] = col < nd + nb * kgs
    s["mean"] = torch.zeros((b, wide), device="cuda") if case["weights"] else None
    if own:
        s["call"] = _shared_call(s)
    return s


def prepare(case, seed):
    return (_prepare_rope if case["kind"] == "rope" else _prepare_shared)(case, _generator(seed))


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _rope_call(s):
    """What a program fills in once: the arguments of tt_qk_norm_rope."""
    from tritiercache_amd import _lib

    case, p = s["case"], lambda k: s[k].data_ptr() if k in s else None
    a = _lib.QkRope()
    for x in ("q", "k", "v", "q_out", "k_out", "v_out"):
        setattr(a, x, p(x))
        setattr(a, x + "_token_stride", s[x].stride(0))
        setattr(a, x + "_head_stride", s[x].stride(1))
    a.q_weight, a.k_weight, a.cos, a.sin, a.positions, a.rows = (p(k) for k in ("qw", "kw", "cos", "sin", "positions",
                                                                                "rows"))
    a.table_rows, a.table_stride, a.out_rows, a.tokens = s["cos"].shape[0], case["rot"], s["out_rows"], case["tokens"]
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.rotary_dim = case["hq"], case["hkv"], case["d"], case["rot"]
    a.eps = 1e-6
    a.in_dtype = a.weight_dtype = CODE[case["src"]]
    a.out_dtype, a.table_dtype = CODE[case["dst"]], CODE[case["table"]]
    return _lib.load(), ctypes.byref(a), a


_TIERS = (("dense_K", "dk"), ("dense_V", "dv"), ("PBS_K_Packed", "kp"), ("PBS_K_Scales", "ks"), ("PBS_K_Zeroes", "kz"),
          ("PBS_V_Packed", "vp"), ("PBS_V_Scales", "vs"), ("PBS_V_Zeroes", "vz"), ("PBS_token_ids", "ids"))


def _shared_call(s):
    """What a serving loop keeps while its tables hold: the sequences' table on host and device, and a workspace."""
    from tritiercache_amd import _lib

    lib, case = _lib.load(), s["case"]
    hq, hkv, d, kgs, b = (case[k] for k in ("hq", "hkv", "d", "kgs", "seqs"))
    prefix, seqs = _lib.DecodeSeq(), (_lib.DecodeSeq * b)()
    for field, k in _TIERS:
        setattr(prefix, field, s["prefix"][k].data_ptr() or None)
        step = s["own"][k].numel() // b * s["own"][k].element_size()
        for i in range(b):
            setattr(seqs[i], field, s["own"][k].data_ptr() + i * step if step else None)
    prefix.dense_count, prefix.num_blocks = s["pd"], s["pb"]
    for i, (nd, nb) in enumerate(s["lengths"]):
        seqs[i].Q, seqs[i].attn_output = s["q"][i].data_ptr(), s["out"][i].data_ptr()
        seqs[i].mean_attn_weights = s["mean"][i].data_ptr() if case["weights"] else None
        seqs[i].dense_count, seqs[i].num_blocks = nd, nb
    table = torch.frombuffer(bytearray(bytes(seqs)), dtype=torch.uint8).cuda()
    size = lib.tt_shared_decode_workspace_bytes(ctypes.byref(prefix), seqs, b, hq, hkv, d, kgs)
    if size == 0:
        _lib.check(_lib.TT_ERR_INVALID_ARGUMENT, "shared")
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    args = (ctypes.byref(prefix), seqs, table.data_ptr(), b, hq, hkv, d, kgs, int(case["meta"] == "fp16"),
            ws.data_ptr(), size)
    return lib, args, (prefix, table, ws)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _run_own(s):
    from tritiercache_amd import _lib

    lib, args, _ = s["call"]
    if s["case"]["kind"] == "rope":
        _lib.check(lib.tt_qk_norm_rope(args, _stream()), "qk_norm_rope")
    else:
        _lib.check(lib.tt_fused_attention_decode_shared(*args, _stream()), "fused_attention_decode_shared")


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _rotated(x, w, cos, sin, rot, eps=1e-6):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()
    y = x[..., :rot]
    turned = torch.cat([-y[..., rot // 2:], y[..., :rot // 2]], -1)
    return torch.cat([y * cos + turned * sin, x[..., rot:]], -1)


def _run_rope(s):
    case = s["case"]
    n, rot = case["tokens"], case["rot"]
    cos, sin = (s[k][s["positions"]] if case["slots"] else s[k][:n] for k in ("cos", "sin"))
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    q, k = (_rotated(s[x], s.get(x + "w"), cos, sin, rot) for x in ("q", "k"))
    s["q_out"].copy_(q)
    rows = torch.where(s["rows"] < 0, s["out_rows"], s["rows"]) if case["slots"] else None
    for out, x in ((s["k_out"], k), (s["v_out"], s["v"])):
        if rows is None:
            out[:n].copy_(x)
        else:
            out.index_copy_(0, rows, x.to(out.dtype))


def _meta(x, case):
    return (x.view(torch.float16) if case["meta"] == "fp16" else x).float()


def _unpacked(t, case):
    """Keys and values [slots, Hkv, D] of packed blocks in 32 bits."""
    hkv, d, kgs = case["hkv"], case["d"], case["kgs"]
    shift = 2 * torch.arange(16, device="cuda", dtype=torch.int32)
    codes = ((t["kp"][:, :, None] >> shift[:, None, None]) & 3).float().view(-1, kgs, hkv, d)
    k = codes * _meta(t["ks"], case)[:, None] + _meta(t["kz"], case)[:, None]
    codes = ((t["vp"][..., None] >> shift) & 3).float().view(-1, hkv, d)
    v = codes * _meta(t["vs"], case)[..., None] + _meta(t["vz"], case)[..., None]
    return k.reshape(-1, hkv, d), v


def _run_shared(s):
    case = s["case"]
    hq, hkv, d, kgs, b = (case[k] for k in ("hq", "hkv", "d", "kgs", "seqs"))
    grp, cd, cb = hq // hkv, case["dense"], case["blocks"]
    k, v = _unpacked(s["prefix"], case)
    k, v = (torch.cat([s["prefix"][n], x]).transpose(0, 1) for n, x in (("dk", k), ("dv", v)))  # [Hkv, P, D]
    hide = torch.cat([s["prefix"]["ids"].new_zeros(s["pd"]), s["prefix"]["ids"]]) == -1
    ok, ov = _unpacked(s["own"], case)
    ok, ov = (torch.cat([s["own"][n].view(b, cd, hkv, d), x.view(b, cb * kgs, hkv, d)], 1).transpose(1, 2)
              for n, x in (("dk", ok), ("dv", ov)))  # [B, Hkv, O, D]
    q = s["q"].view(b, hkv, grp, d) / math.sqrt(d)
    qp = q.transpose(0, 1).reshape(hkv, b * grp, d)
    sp = (qp @ k.transpose(1, 2)).masked_fill(hide, -math.inf)  # [Hkv, B G, P]
    so = (q @ ok.transpose(2, 3)).masked_fill(~s["live"][:, None, None], -math.inf)  # [B, Hkv, G, O]
    m = torch.maximum(sp.amax(-1).view(hkv, b, grp).transpose(0, 1), so.amax(-1))
    pp = torch.exp(sp - m.transpose(0, 1).reshape(hkv, b * grp, 1))
    po = torch.exp(so - m[..., None])
    total = pp.sum(-1).view(hkv, b, grp).transpose(0, 1) + po.sum(-1)
    out = (pp @ v).view(hkv, b, grp, d).transpose(0, 1) + po @ ov
    s["out"].copy_((out / total[..., None]).reshape(b, hq, d))
    if case["weights"]:
        w = (po / total[..., None]).mean((1, 2))
        s["mean"].copy_(w.gather(1, s["column"]) * s["used"])


def run(s):
    if own:
        _run_own(s)
    else:
        (_run_rope if s["case"]["kind"] == "rope" else _run_shared)(s)
    if s["case"]["kind"] == "rope":
        return [s["q_out"], s["k_out"][:s["out_rows"]], s["v_out"][:s["out_rows"]]]
    return [s["out"], s["mean"]] if s["case"]["weights"] else [s["out"]]


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope(s):
    case = s["case"]
    n, d, rot, half = case["tokens"], case["d"], case["rot"], case["rot"] // 2
    at = s["positions"] if case["slots"] else torch.arange(n, device="cuda")
    cos, sin = s["cos"].double()[at], s["sin"].double()[at]
    got = []
    for name in ("q", "k"):
        x = s[name].double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * s[name + "w"].double()
        y = x.clone()
        y[..., :half] = x[..., :half] * cos[:, None, :half] - x[..., half:rot] * sin[:, None, :half]
        y[..., half:rot] = x[..., half:rot] * cos[:, None, half:] + x[..., :half] * sin[:, None, half:]
        got.append(y)
    q, k = got
    if not case["slots"]:
        return [q, k, s["v"].double()]
    kept = s["rows"] >= 0
    tiers = []
    for x in (k, s["v"].double()):
        t = torch.zeros((s["out_rows"],) + tuple(x.shape[1:]), dtype=torch.float64, device="cuda")
        t[s["rows"][kept]] = x[kept]
        tiers.append(t)
    return [q] + tiers


def _tokens64(t, case, dense, block0, blocks, dense0=0):
    """Keys and values [tokens, Hkv, D] of `dense` FP32 rows and `blocks` blocks in 64 bits, and which are attended."""
    hkv, d, kgs = case["hkv"], case["d"], case["kgs"]
    real = lambda x: x.view(torch.float16).double() if x.dtype == torch.uint16 else x.double()  # noqa: E731
    b, n = slice(block0, block0 + blocks), slice(block0 * kgs, (block0 + blocks) * kgs)
    kp, vp = t["kp"][b].long() & 0xFFFFFFFF, t["vp"][n].long() & 0xFFFFFFFF
    kc = torch.stack([(kp >> (2 * i)) & 3 for i in range(16)], 2).reshape(blocks, kgs, hkv, d)
    vc = torch.stack([(vp >> (2 * i)) & 3 for i in range(16)], 3).reshape(blocks * kgs, hkv, d)
    k = (kc * real(t["ks"][b]).unsqueeze(1) + real(t["kz"][b]).unsqueeze(1)).reshape(-1, hkv, d)
    v = vc * real(t["vs"][n]).unsqueeze(-1) + real(t["vz"][n]).unsqueeze(-1)
    seen = torch.cat([torch.ones(dense, dtype=torch.bool, device="cuda"), t["ids"].reshape(-1)[n] >= 0])
    r = slice(dense0, dense0 + dense)
    return torch.cat([t["dk"][r].double(), k]), torch.cat([t["dv"][r].double(), v]), seen


def _exact_shared(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    grp = hq // hkv
    pk, pv, pseen = _tokens64(s["prefix"], case, s["pd"], 0, s["pb"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    mean = torch.zeros(s["mean"].shape, dtype=torch.float64, device="cuda") if case["weights"] else None
    for i, (nd, nb) in enumerate(s["lengths"]):
        k, v, seen = _tokens64(s["own"], case, nd, i * case["blocks"], nb, i * case["dense"])
        for j in range(hkv):
            q = s["q"][i, j * grp:(j + 1) * grp].double()
            x = torch.cat([q @ pk[:, j].T, q @ k[:, j].T], 1) / math.sqrt(d)
            x[:, ~torch.cat([pseen, seen])] = -math.inf
            p = torch.softmax(x, 1)
            n = pk.shape[0]
            out[i, j * grp:(j + 1) * grp] = p[:, :n] @ pv[:, j] + p[:, n:] @ v[:, j]
            if mean is not None:
                mean[i, :k.shape[0]] += p[:, n:].sum(0) / hq
    return [out] if mean is None else [out, mean]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rope(s) if case["kind"] == "rope" else _exact_shared(s)
