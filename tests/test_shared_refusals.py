"""What tt_fused_attention_decode_shared refuses, on the CPU: every rejected call returns before any launch (the
pointers are placeholders, never dereferenced)."""
import ctypes as C
import random

import pytest

_lib = pytest.importorskip("tritiercache_amd._lib")

P = 0x100000
TIERS = ("dense_K", "dense_V", "PBS_K_Packed", "PBS_K_Scales", "PBS_K_Zeroes", "PBS_V_Packed", "PBS_V_Scales",
         "PBS_V_Zeroes", "PBS_token_ids")


def tables(n=3, prefix=(40, 7), own=(5, 2)):
    p, s = _lib.DecodeSeq(), (_lib.DecodeSeq * n)()
    for x, (nd, nb) in [(p, prefix)] + [(x, own) for x in s]:
        for f in TIERS:
            setattr(x, f, P)
        x.dense_count, x.num_blocks = nd, nb
    for x in s:
        x.Q, x.attn_output = P, P
    return p, s


def call(p, s, n=None, hq=8, hkv=2, d=128, kgs=16, dev=P, ws=P, size=1 << 40):
    L = _lib.load()
    return L.tt_fused_attention_decode_shared(C.byref(p) if p is not None else None, s, dev, len(s) if n is None else n,
                                              hq, hkv, d, kgs, 0, ws, size, None)


@pytest.mark.parametrize("kw,word", [({"n": -1}, "num_seqs"), ({"hq": 7}, "multiple"), ({"d": 72}, "head_dim"),
                                     ({"d": 272}, "head_dim"), ({"kgs": 24}, "k_group_size"), ({"hkv": 0}, ""),
                                     ({"dev": None}, "seqs_device"), ({"ws": None}, "workspace"),
                                     ({"size": 1000}, "workspace")], ids=str)
def test_shapes_and_workspace(kw, word):
    p, s = tables()
    assert call(p, s, **kw) == _lib.TT_ERR_INVALID_ARGUMENT and word in _lib.last_error(), _lib.last_error()


def test_prefix_and_sequences():
    p, s = tables()
    assert call(None, s) == 1 and "prefix" in _lib.last_error()
    for f in TIERS:
        p, s = tables()
        setattr(p, f, None)
        assert call(p, s) == 1, f
        p, s = tables()
        setattr(s[1], f, None)
        assert call(p, s) == 1, f
    for f in ("Q", "attn_output"):
        p, s = tables()
        setattr(s[2], f, None)
        assert call(p, s) == 1 and f in _lib.last_error()
    p, s = tables()
    p.mean_attn_weights = P
    assert call(p, s) == 1 and "mean" in _lib.last_error()
    for f in ("dense_count", "num_blocks"):
        for which in (0, 1):
            p, s = tables()
            setattr((p, s[1])[which], f, -1)
            assert call(p, s) == 1 and f in _lib.last_error()
    p, s = tables(prefix=(1 << 30, 1 << 27))
    assert call(p, s) == 1 and "2^31" in _lib.last_error()
    p, s = tables()
    s[0].dense_count, s[0].mean_attn_weights = 1 << 28, P
    assert call(p, s) == 1 and "4 GiB" in _lib.last_error()
    p, s = tables()
    assert call(p, s, n=0) == _lib.TT_OK  # nothing to do


def test_the_size_query_validates_and_every_sized_call_is_accepted():
    """Without a device an accepted call ends at its launch; with one it would run on the placeholders."""
    L = _lib.load()
    p, s = tables()
    assert L.tt_shared_decode_workspace_bytes(C.byref(p), s, 3, 7, 2, 128, 16) == 0 and _lib.last_error()
    assert L.tt_shared_decode_workspace_bytes(None, s, 3, 8, 2, 128, 16) == 0
    if L.tt_device_count() > 0:
        pytest.skip("placeholder pointers: only where no kernel can run")
    rng = random.Random(3)
    for _ in range(1500):
        n = rng.choice((1, 2, 7, 33, 64, 65, 130))
        pre = (rng.choice((0, 1, 300, 4000)), int(10 ** rng.uniform(0, 4)) - 1)
        p, s = tables(n, pre)
        for x in s:
            x.dense_count, x.num_blocks = rng.randint(0, 300), rng.choice((0, 0, 5, 400))
            x.mean_attn_weights = rng.choice((None, P))
        hkv, g = rng.choice((1, 2, 3, 8, 32)), rng.choice((1, 2, 3, 4, 7, 8, 17))
        d, kgs = 16 * rng.randint(1, 16), rng.choice((16, 32))
        size = L.tt_shared_decode_workspace_bytes(C.byref(p), s, n, hkv * g, hkv, d, kgs)
        assert size > 0, _lib.last_error()
        rc = L.tt_fused_attention_decode_shared(C.byref(p), s, P, n, hkv * g, hkv, d, kgs, 0, P, size, None)
        assert rc == _lib.TT_ERR_HIP, (rc, _lib.last_error())


def test_python_form():
    from tritiercache_amd import _C

    with pytest.raises(ValueError):
        _C.fused_attention_decode_shared({"mean_attn_weights": 1}, [], 8, 2, 128)
    with pytest.raises(ValueError):
        _C.fused_attention_decode_shared({}, [], 8, 0, 128)


def test_a_tensor_that_is_too_small_is_refused():
    torch = pytest.importorskip("torch")
    from tritiercache_amd import _C

    st = _C._Staging(sized=True)
    with pytest.raises(ValueError, match="'Q' tensor holds 12 bytes, the call needs 16"):
        st.ptr(torch.zeros(3), "Q", 16)
    with pytest.raises(ValueError, match="'PBS_K_Scales'"):
        st.ptr(torch.zeros(8, dtype=torch.float16), "PBS_K_Scales", 32)  # FP16 metadata behind an FP32 call


@pytest.mark.gpu
def test_too_small_tensors_and_prefixes_with_weights_on_the_gpu():
    torch = pytest.importorskip("torch")
    from tritiercache_amd import _C

    def seq(**kw):
        e = {"Q": torch.zeros((8, 64), device="cuda"), "attn_output": torch.full((8, 64), 7.0, device="cuda"),
             "dense_K": torch.zeros((2, 2, 64), device="cuda"), "dense_V": torch.zeros((2, 2, 64), device="cuda"),
             "dense_count": 2, "num_blocks": 0}
        return {**e, **kw}

    pre = {k: v for k, v in seq().items() if k not in ("Q", "attn_output")}
    for bad in ({"Q": torch.zeros((7, 64), device="cuda")}, {"attn_output": torch.zeros(8, 63, device="cuda")},
                {"dense_count": 3}, {"Q": torch.zeros((8, 64), dtype=torch.float16, device="cuda")},
                {"mean_attn_weights": torch.zeros(1, device="cuda")}):
        good = seq()
        with pytest.raises(ValueError, match="tensor holds"):
            _C.fused_attention_decode_shared(pre, [good, seq(**bad)], 8, 2, 64)
        torch.cuda.synchronize()
        assert bool((good["attn_output"] == 7).all())
    with pytest.raises(ValueError, match="tensor holds"):
        _C.fused_attention_decode_shared({**pre, "dense_count": 9}, [seq()], 8, 2, 64)
    with pytest.raises(ValueError, match="mean attention weights"):
        _C.fused_attention_decode_shared({**pre, "mean_attn_weights": torch.zeros(2, device="cuda")}, [seq()], 8, 2, 64)
    good = seq()
    _C.fused_attention_decode_shared(pre, [good], 8, 2, 64)
    torch.cuda.synchronize()
    assert bool((good["attn_output"] == 0).all())
