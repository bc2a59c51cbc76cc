"""What tt_qk_norm_rope and its Python form refuse, on the CPU: every rejected call returns before any launch (the
pointers are placeholders, never dereferenced)."""
import ctypes as C

import pytest
import torch

_lib = pytest.importorskip("tritiercache_amd._lib")

P = 0x100000


def args(**kw):
    a = _lib.QkRope()
    t, hq, hkv, d = 6, 4, 2, 64
    for i, n in enumerate(("q", "k", "v", "q_out", "k_out", "v_out", "cos", "sin", "positions", "rows")):
        setattr(a, n, P + (i << 20))
    for n, h in (("q", hq), ("k", hkv), ("v", hkv)):
        for s in (n, n + "_out"):
            setattr(a, s + "_token_stride", h * d)
            setattr(a, s + "_head_stride", d)
    a.tokens, a.num_q_heads, a.num_kv_heads, a.head_dim, a.rotary_dim = t, hq, hkv, d, d
    a.table_rows, a.table_stride, a.out_rows, a.eps = 100, d, 20, 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    return a


REFUSED = [
    ({"tokens": -1}, "tokens"), ({"num_q_heads": 0}, "num_q_heads"), ({"num_kv_heads": -2}, "num_kv_heads"),
    ({"head_dim": 0}, "head_dim"), ({"head_dim": 72}, "head_dim"), ({"head_dim": 272}, "head_dim"),
    ({"rotary_dim": 8}, "rotary_dim"), ({"rotary_dim": 80}, "rotary_dim"), ({"rotary_dim": -16}, "rotary_dim"),
    ({"in_dtype": 3}, "dtype"), ({"out_dtype": -1}, "dtype"), ({"weight_dtype": 7}, "dtype"),
    ({"table_dtype": 4}, "dtype"), ({"eps": -1e-6}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"q_token_stride": -1}, "strides"), ({"v_head_stride": -64}, "strides"),
    ({"q": None}, "'q'"), ({"k_out": None}, "'k_out'"), ({"v": None}, "v_out"), ({"v_out": None}, "v_out"),
    ({"cos": None}, "'cos'"), ({"sin": None}, "'sin'"), ({"table_stride": 63}, "table_stride"),
    ({"positions": None, "table_rows": 5}, "tables"), ({"rows": None, "out_rows": 5}, "out_rows"),
    ({"q_out_head_stride": 63}, "overlap"), ({"q_out_token_stride": 255}, "overlap"),
    ({"k_out_token_stride": 0}, "overlap"), ({"v_out_head_stride": 0}, "overlap"),
    ({"q_out": P, "q_out_token_stride": 512}, "place"), ({"q_out": P, "out_dtype": 1}, "place"),
    ({"k_out": P + (1 << 20)}, "place"),  # rows are given
]


@pytest.mark.parametrize("change,word", REFUSED, ids=str)
def test_refused(change, word):
    L = _lib.load()
    assert L.tt_qk_norm_rope(C.byref(args(**change)), None) == _lib.TT_ERR_INVALID_ARGUMENT
    assert word in _lib.last_error(), _lib.last_error()


def test_no_arguments_and_no_tokens():
    L = _lib.load()
    assert L.tt_qk_norm_rope(None, None) == _lib.TT_ERR_INVALID_ARGUMENT
    a = args(tokens=0, q=None, k=None, v=None, q_out=None, k_out=None, v_out=None, cos=None, sin=None)
    assert L.tt_qk_norm_rope(C.byref(a), None) == _lib.TT_OK  # nothing to do, nothing launched


def test_accepted_strides_reach_the_launch():
    """Heads inside tokens, tokens inside heads (a transposed output) and rows of a joint buffer are accepted: without
    a device they end at the launch."""
    L = _lib.load()
    if L.tt_device_count() > 0:
        pytest.skip("placeholder pointers: only where no kernel can run")
    for kw in ({}, {"q_out_token_stride": 64, "q_out_head_stride": 6 * 64}, {"q_token_stride": 8 * 64},
               {"k_out_token_stride": 1000}, {"v": None, "v_out": None}, {"rotary_dim": 0, "cos": None, "sin": None},
               {"q_out": P, "in_dtype": 2, "out_dtype": 2}, {"positions": None}, {"rows": None}):
        assert L.tt_qk_norm_rope(C.byref(args(**kw)), None) == _lib.TT_ERR_HIP, (kw, _lib.last_error())


def test_python_form_refuses_before_it_needs_a_gpu():
    from tritiercache_amd import _C

    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    cos = torch.zeros(8, 64)
    for kw in (dict(v=torch.zeros(3, 4, 64)), dict(v=torch.zeros(2, 2, 64)), dict(cos=cos), dict(sin=cos),
               dict(cos=cos, sin=torch.zeros(8, 32)), dict(cos=cos, sin=cos, positions=torch.zeros(3)),
               dict(cos=cos, sin=cos, positions=torch.zeros(2, dtype=torch.int64)), dict(q_weight=torch.ones(32)),
               dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.float16)),
               dict(rows=torch.zeros(3, dtype=torch.int64)), dict(v_out=k), dict(positions=[0, 1, 2])):
        with pytest.raises(ValueError):
            _C.qk_norm_rope(q, k, **kw)
    for bad in (q.double(), q[..., ::2], q[0], [1]):
        with pytest.raises(ValueError):
            _C.qk_norm_rope(bad, k)


def test_struct_layout_matches_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    names = [f[0] for f in _lib.QkRope._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tritiercache_amd.h"\nint main(void) {\n'
                   '  printf("%zu\\n", sizeof(tt_qk_rope));\n'
                   + "".join(f'  printf("%zu\\n", offsetof(tt_qk_rope, {n}));\n' for n in names) + "  return 0;\n}\n")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [C.sizeof(_lib.QkRope)] + [getattr(_lib.QkRope, n).offset for n in names]


def test_inputs_that_record_gradients_are_refused():
    from tritiercache_amd import _C

    q, k, w = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.ones(64)
    for name in ("q", "k", "v", "q_weight", "q_out"):
        given = {"q": q, "k": k, "v": k.clone(), "q_weight": w, "q_out": q.clone()}
        given[name] = given[name].clone().requires_grad_()
        with pytest.raises(ValueError, match="no backward pass"):
            _C.qk_norm_rope(**given)
