"""The operators of a decode step behind a shared prompt, together: the prompt through qk_norm_rope into a
TriTierCache, its tiers as the prefix of a batch (as_prefix), and steps of the batch whose keys and values
qk_norm_rope appends to the sequences' tiers and fused_attention_decode_shared reads. Each operator's outputs are
checked against its formula in 64 bits over the inputs that it got, within its own tolerance. And the patch's
FUSED_QK path against the model file's modules."""
import pytest
import torch

from test_gpu_qk_rope import check as check_qk
from test_gpu_qk_rope import formula, tables
from test_gpu_shared import check as check_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def C():
    from tritiercache_amd import _C

    return _C


def _cache(hq, hkv, d, kgs, meta):
    from tritiercache_amd.cache import TriTierCache

    return TriTierCache(max_seq_len=2048, head_dim=d, num_heads=hkv, R_size=64, H_ratio=0.05, num_q_heads=hq,
                        k_group_size=kgs, pbs_metadata_dtype=meta)


@pytest.mark.parametrize("prompt", [0, 1, 3, 50, 68, 69, 500])
@pytest.mark.parametrize("kgs,meta", [(16, "fp16"), (32, "fp32")])
def test_as_prefix_holds_what_the_next_step_attends_to(C, prompt, kgs, meta):
    hq, hkv, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(prompt)
    c = _cache(hq, hkv, d, kgs, meta)
    if prompt:
        c.prefill(*(torch.randn((prompt, hkv, d), generator=g, device="cuda") for _ in range(2)))
        for _ in range(5):  # moves the ring's head
            x = [torch.randn(h * d, generator=g, device="cuda") for h in (hq, hkv, hkv)]
            c.step(*x, torch.empty(hq * d, device="cuda"))
    p = c.as_prefix()
    K, V, ids = c.reconstruct_full_cache()
    s, hh, rw = c.S_count, c.HH_count, c.RW_count
    nb = p["num_blocks"]
    assert p["dense_count"] == s + hh + rw == p["dense_K"].shape[0] == p["dense_V"].shape[0]
    pk = torch.empty((nb * kgs, hkv, d), device="cuda")
    pv = torch.empty_like(pk)
    if nb:
        C.dequantize_k(p["PBS_K_Packed"], p["PBS_K_Scales"], p["PBS_K_Zeroes"], pk, nb, hkv, d, kgs, meta)
        C.dequantize_v(p["PBS_V_Packed"], p["PBS_V_Scales"], p["PBS_V_Zeroes"], pv, nb * kgs, hkv, d, meta)
        keep = p["PBS_token_ids"] != -1
        pk, pv = pk[keep], pv[keep]
    for got, want in ((torch.cat([p["dense_K"], pk]), K), (torch.cat([p["dense_V"], pv]), V)):
        assert torch.equal(got[:s], want[:s])
        assert torch.equal(got[s + hh:s + hh + rw], want[want.shape[0] - rw:])  # oldest first
        assert torch.equal(got.flatten(1).sort(0)[0], want.flatten(1).sort(0)[0])
    if prompt:  # later calls leave the copies as they are
        before = {k: v.clone() for k, v in p.items() if isinstance(v, torch.Tensor)}
        for _ in range(40):
            x = [torch.randn(h * d, generator=g, device="cuda") for h in (hq, hkv, hkv)]
            c.step(*x, torch.empty(hq * d, device="cuda"))
        assert all(torch.equal(p[k], v) for k, v in before.items())


@pytest.mark.parametrize("hq,hkv,d,b,prompt,kgs,meta", [(8, 2, 128, 5, 900, 16, "fp16"), (8, 2, 128, 40, 700, 32, "fp32"),
                                                        (6, 6, 80, 36, 600, 16, "fp32"), (4, 1, 64, 1, 300, 16, "fp16")])
def test_a_batch_behind_a_shared_prompt(C, hq, hkv, d, b, prompt, kgs, meta):
    g = torch.Generator(device="cuda").manual_seed(b)
    steps, cap = 5, 8
    cos, sin = tables(prompt + steps, d, torch.float32, g)
    wq, wk = ((1 + torch.randn(d, generator=g, device="cuda") / 4).to(BF16) for _ in range(2))

    def projected(tokens):  # one joint projection's q, k and v
        x = torch.randn((tokens, hq + 2 * hkv, d), generator=g, device="cuda").to(BF16)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    def verify(x, w, got, pos, tag):
        check_qk(got, *formula(x, w, cos[pos], sin[pos], 1e-6), tag)

    q, k, v = projected(prompt)
    _, pk, pv = C.qk_norm_rope(q, k, v, cos[:prompt], sin[:prompt], q_weight=wq, k_weight=wk, out_dtype=torch.float32)
    verify(k, wk, pk, torch.arange(prompt, device="cuda"), "prompt")
    assert torch.equal(pv, v.float())
    cache = _cache(hq, hkv, d, kgs, meta)
    cache.prefill(pk, pv)
    prefix = cache.as_prefix()
    assert prefix["num_blocks"] > 0
    K, V, _ = cache.reconstruct_full_cache()
    ref = (K.double(), V.double(), torch.ones(K.shape[0], dtype=torch.bool, device="cuda"))

    own_k = torch.full((b * cap, hkv, d), float("nan"), device="cuda")
    own_v = torch.full_like(own_k, float("nan"))
    out = torch.empty((b, hq, d), device="cuda")
    for t in range(steps):
        q, k, v = projected(b)
        rows = torch.arange(b, device="cuda") * cap + t
        pos = torch.full((b,), prompt + t, dtype=torch.int64, device="cuda")
        kept = own_k.clone()
        qr, _, _ = C.qk_norm_rope(q, k, v, cos, sin, positions=pos, q_weight=wq, k_weight=wk, rows=rows, k_out=own_k,
                                  v_out=own_v, out_dtype=torch.float32)
        verify(q, wq, qr, pos, ("q", t))
        verify(k, wk, own_k[rows], pos, ("k", t))
        assert torch.equal(own_v[rows], v.float())
        kept[rows] = own_k[rows]
        assert torch.equal(kept.view(torch.int32), own_k.view(torch.int32))  # no other row
        batch = [{"Q": qr[i], "dense_K": own_k[i * cap:i * cap + t + 1], "dense_V": own_v[i * cap:i * cap + t + 1],
                  "dense_count": t + 1, "num_blocks": 0, "attn_output": out[i],
                  "mean_attn_weights": torch.empty(t + 1, device="cuda")} for i in range(b)]
        C.fused_attention_decode_shared(prefix, batch, hq, hkv, d, kgs, meta)
        all_valid = torch.ones(t + 1, dtype=torch.bool, device="cuda")
        for i in range(b):
            own = (batch[i]["dense_K"].double(), batch[i]["dense_V"].double(), all_valid)
            check_attention(out[i], batch[i]["mean_attn_weights"], qr[i], ref, own, hkv, (t, i))


# ---------------------------------------------------------------------------
# The patch with FUSED_QK
# ---------------------------------------------------------------------------
transformers = pytest.importorskip("transformers")


@pytest.fixture
def fused(monkeypatch):
    """The patch, with a count of the fused launches."""
    from tritiercache_amd.integration import patch_model

    calls = []
    real = patch_model._C.qk_norm_rope
    monkeypatch.setattr(patch_model._C, "qk_norm_rope", lambda *a, **k: calls.append(a[0].shape[0]) or real(*a, **k))
    monkeypatch.setattr(patch_model, "FUSED_QK", True)
    patch_model.apply_patch()
    yield patch_model, calls
    patch_model.remove_patch()


def _attention(arch, dtype, d=64):
    import transformers as tf

    if arch == "qwen3":
        from transformers.models.qwen3.modeling_qwen3 import Qwen3Attention as A
        cfg = tf.Qwen3Config(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=d)
    else:
        from transformers.models.llama.modeling_llama import LlamaAttention as A
        cfg = tf.LlamaConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=d)
    torch.manual_seed(5)
    layer = A(cfg, layer_idx=0).to("cuda", dtype)
    if arch == "qwen3":
        with torch.no_grad():
            for w in (layer.q_norm.weight, layer.k_norm.weight):
                w.add_(torch.randn_like(w) / 4)
    return layer, cfg


@pytest.mark.parametrize("arch", ["llama", "qwen3"])
@pytest.mark.parametrize("dtype", [torch.float32, BF16, torch.float16])
@pytest.mark.parametrize("n", [1, 37])
def test_fused_qk_against_the_modules(fused, arch, dtype, n):
    """Both paths against 64 bits differ by their roundings alone. The fused one's: see test_gpu_qk_rope. The modules'
    round to the type (e: half a step, relative) behind the norm, its weight, either product and the sum: at most
    2 e + e of |y c| + |y' s| and e of the result, e^2 terms under e/8 of it, besides FP32's 20 half steps."""
    patch_model, calls = fused
    layer, cfg = _attention(arch, dtype)
    d = cfg.head_dim
    g = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn((1, n, cfg.hidden_size), generator=g, device="cuda").to(dtype)
    a = torch.rand((1, n, d // 2), generator=g, device="cuda") * 6.3
    pos = tuple(torch.cat([x, x], -1).to(dtype) for x in (a.cos(), a.sin()))
    with torch.no_grad():
        got = patch_model._rotated_qkv(layer, h, pos)
        assert calls == [n]
        patch_model.FUSED_QK = False
        want = patch_model._rotated_qkv(layer, h, pos)
        assert calls == [n]
        e = torch.finfo(dtype).eps / 2
        for i, name in ((0, "q"), (1, "k")):
            x = getattr(layer, name + "_proj")(h).view(n, -1, d)
            w = getattr(layer, name + "_norm").weight if arch == "qwen3" else None
            z, mag = formula(x, w, pos[0][0], pos[1][0], 1e-6)
            z, mag = z.transpose(0, 1)[None], mag.transpose(0, 1)[None]
            assert got[i].shape == want[i].shape and got[i].dtype == (torch.float32 if n == 1 else dtype)
            tiny = torch.finfo(dtype).smallest_normal * e * 4
            off = (got[i].double() - want[i].double()).abs()
            bound = e * (3.125 * mag + 2 * z.abs()) + 40 * 2.0 ** -24 * mag + tiny
            assert bool((off <= bound).all()), float((off / bound).max())
        assert torch.equal(got[2].to(dtype), want[2])


def test_fused_qk_in_a_forward(fused):
    """A prompt and decode tokens through the patched layer, one fused launch each; none where gradients are recorded or
    a norm has a hook, where the modules run as before."""
    patch_model, calls = fused
    for arch in ("llama", "qwen3"):
        layer, cfg = _attention(arch, BF16)
        del calls[:]

        def forward(n, first, **kw):
            h = torch.randn((1, n, cfg.hidden_size), device="cuda", dtype=BF16)
            a = torch.arange(first, first + n, device="cuda")[:, None] / 100 ** torch.rand(cfg.head_dim // 2, device="cuda")
            pos = tuple(torch.cat([x, x], -1)[None].to(BF16) for x in (a.cos(), a.sin()))
            out, w = layer(h, position_embeddings=pos, **kw)
            assert out.shape == h.shape and out.dtype == BF16 and torch.isfinite(out).all()
            return w

        with torch.no_grad():
            forward(20, 0)
            forward(1, 20)
            assert forward(1, 21, output_attentions=True).shape == (1, 4, 1, 22)
        assert calls == [20, 1, 1] and layer.tri_tier_cache.Total_Processed_Tokens == 22
        forward(3, 22)  # records gradients
        assert calls == [20, 1, 1]
        if arch == "qwen3":
            handle = layer.k_norm.register_forward_hook(lambda m, x, y: y)
            with torch.no_grad():
                forward(1, 25)
                assert calls == [20, 1, 1]
                handle.remove()
                forward(1, 26)
            assert calls == [20, 1, 1, 1]


def test_fused_qk_generate(fused):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    patch_model, calls = fused
    cfg = Qwen3Config(vocab_size=100, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=16, max_position_embeddings=256, pad_token_id=0, bos_token_id=1,
                      eos_token_id=2)
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to("cuda").eval()
    with torch.no_grad():
        out = model.generate(torch.tensor([[1, 5, 7]], device="cuda"), max_new_tokens=12, use_cache=True, eos_token_id=None,
                             do_sample=False)
    assert out.shape == (1, 15)
    assert calls == [3, 3] + [1] * 22
