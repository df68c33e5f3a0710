"""Calls that the cache, norm-and-rotation and attention operators refuse before anything reaches the device (no GPU: the
check for a CUDA device comes last)."""
import pytest
import torch

from triteia_b200 import _lib, capi, ops

H, D, P, PAGES = 2, 64, 16, 4


def test_cpu_tensors_are_rejected():
    kc, vc, _, _ = ops.new_cache(PAGES, P, H, D, device="cpu")
    x, slots = torch.zeros(3, H, D, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cache_write(x, x, kc, vc, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cache_read(kc, vc, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(x, kc, vc, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        capi.qk_norm_rotary_embedding(slots, x.view(3, -1), x.view(3, -1), D, torch.zeros(8, D, dtype=torch.float16), True)


def _attention(**change):
    """trb_paged_attention with a good set of arguments but for `change`; the pointers are never read: every call that is
    made here is refused on the host."""
    a = dict(query=64, key_cache=64, value_cache=64, key_exponents=None, value_exponents=None, page_table=64, lengths=64, query_starts=64,
             out=64, num_tokens=3, num_seqs=2, num_heads=4, num_kv_heads=2, head_size=64, page_size=16, num_pages=4, table_stride=2,
             table_width=2, query_token_stride=256, query_head_stride=64, out_token_stride=256, out_head_stride=64, page_stride=2048,
             token_stride=128, head_stride=64, exp_page_stride=0, exp_token_stride=0, exp_head_stride=0, scale=0.125, causal=1, window=0,
             dtype=0, workspace=64, workspace_bytes=1 << 30, dev=0, stream=None)
    assert set(change) <= set(a)
    return _lib.lib.trb_paged_attention(*{**a, **change}.values())


@pytest.mark.parametrize("change,code", [
    (dict(query=None), 3), (dict(key_cache=None), 3), (dict(value_cache=None), 3), (dict(lengths=None), 3), (dict(out=None), 3),
    (dict(page_table=None), 3), (dict(key_exponents=64), 3), (dict(value_exponents=64), 3), (dict(num_tokens=-1), 3),
    (dict(num_seqs=-1), 3), (dict(num_heads=0), 3), (dict(num_kv_heads=0), 3), (dict(page_size=0), 3), (dict(num_pages=-1), 3),
    (dict(table_width=-1), 3), (dict(window=-1), 3), (dict(query_starts=None), 3),
    (dict(num_heads=5), 1), (dict(window=4, causal=0), 1), (dict(query=72), 1), (dict(out=72), 1), (dict(key_cache=72), 1),
    (dict(value_cache=66), 1), (dict(workspace=72), 1), (dict(query_token_stride=257), 1), (dict(out_head_stride=66), 1), (dict(token_stride=132), 1),
    (dict(table_width=1 << 28, page_size=64), 1), (dict(num_tokens=1 << 30, num_heads=8), 1),
    (dict(head_size=80), 2), (dict(head_size=256), 2), (dict(dtype=2), 2),
])
def test_attention_refuses_on_the_host(change, code):
    assert _attention(**change) == code


def test_attention_without_tokens_or_sequences_does_nothing():
    assert _attention(num_tokens=0) == 0
    assert _attention(num_seqs=0) == 0


def _write(**change):
    a = dict(key=64, value=64, slots=64, key_cache=64, value_cache=64, key_exponents=None, value_exponents=None, num_tokens=3, heads=2,
             head_size=64, page_size=16, num_pages=4, key_token_stride=128, key_head_stride=64, value_token_stride=128,
             value_head_stride=64, page_stride=2048, token_stride=128, head_stride=64, exp_page_stride=0, exp_token_stride=0,
             exp_head_stride=0, dtype=0, dev=0, stream=None)
    return _lib.lib.trb_cache_write(*{**a, **change}.values())


@pytest.mark.parametrize("change,code", [
    (dict(key=None), 3), (dict(value=None), 3), (dict(slots=None), 3), (dict(key_cache=None), 3), (dict(value_cache=None), 3),
    (dict(key_exponents=64), 3), (dict(num_tokens=-1), 3), (dict(heads=0), 3), (dict(page_size=0), 3), (dict(num_pages=-1), 3),
    (dict(head_size=60), 1), (dict(head_size=264), 1), (dict(key=72), 1), (dict(value_cache=72), 1), (dict(key_token_stride=132), 1),
    (dict(value_head_stride=65), 1), (dict(head_stride=68), 1), (dict(dtype=5), 2),
])
def test_cache_write_refuses_on_the_host(change, code):
    assert _write(**change) == code


def _norm(**change):
    a = dict(positions=64, query=64, query_out=64, key=64, key_out=64, query_weight=64, key_weight=64, table=64, cache_is_f32=0,
             max_position=8, num_tokens=3, rot_dim=64, query_stride=128, query_out_stride=128, key_stride=64, key_out_stride=64,
             num_heads=2, num_kv_heads=1, head_size=64, eps=1e-6, is_neox=1, dtype=0, dev=0, stream=None)
    return _lib.lib.trb_qk_norm_rotary(*{**a, **change}.values())


@pytest.mark.parametrize("change,code", [
    (dict(positions=None), 3), (dict(query=None), 3), (dict(query_out=None), 3), (dict(key=None), 3), (dict(key_out=None), 3),
    (dict(table=None), 3), (dict(num_tokens=-1), 3), (dict(num_heads=0), 3), (dict(num_kv_heads=-1), 3), (dict(max_position=-1), 3),
    (dict(head_size=60, rot_dim=60), 1), (dict(head_size=264), 1), (dict(rot_dim=63), 1), (dict(rot_dim=66), 1), (dict(query=72), 1),
    (dict(key_out=72), 1), (dict(query_stride=132), 1), (dict(key_stride=65), 1), (dict(dtype=3), 2),
])
def test_norm_and_rotation_refuse_on_the_host(change, code):
    assert _norm(**change) == code


def test_norm_and_rotation_of_no_tokens_do_nothing():
    assert _norm(num_tokens=0) == 0


def _cache(quantised=False):
    return ops.new_cache(PAGES, P, H, D, device="cpu", quantised=quantised)


SLOTS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("spoil,what", [
    (lambda c: (c[0], c[1][:-1], c[2], c[3]), "same strides"),
    (lambda c: (c[0], c[1].transpose(1, 2).contiguous().transpose(1, 2), c[2], c[3]), "same strides"),
    (lambda c: (c[0].to(torch.float32), c[1].to(torch.float32), c[2], c[3]), "the cache holds"),
    (lambda c: (c[0], c[1], torch.zeros(PAGES, P, H, dtype=torch.uint8), None), "go together"),
    (lambda c: (c[0][..., ::2], c[1][..., ::2], c[2], c[3]), "contiguous last dimension"),
    (lambda c: (c[0][:, :0], c[1][:, :0], c[2], c[3]), "page size"),
    (lambda c: (c[0][0], c[1][0], c[2], c[3]), "same strides"),
])
def test_caches_that_do_not_fit_are_refused(spoil, what):
    kc, vc, ke, ve = spoil(_cache())
    x = torch.zeros(3, H, D, dtype=torch.float16)
    for call in (lambda: ops.cache_write(x, x, kc, vc, SLOTS, ke, ve), lambda: ops.cache_read(kc, vc, SLOTS, ke, ve, dtype=torch.float16),
                 lambda: ops.paged_attention(x, kc, vc, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32), key_exponents=ke,
                                             value_exponents=ve)):
        with pytest.raises(RuntimeError, match=what):
            call()


@pytest.mark.parametrize("spoil,what", [
    (lambda c: c, "CUDA"),
    (lambda c: (c[0], c[1], c[2], None), "go together"),
    (lambda c: (c[0], c[1], None, None), "the cache holds"),
    (lambda c: (c[0], c[1], c[2].int(), c[3].int()), "uint8"),
    (lambda c: (c[0], c[1], c[2][:1], c[3][:1]), "uint8"),
    (lambda c: (c[0], c[1], c[2], c[3].transpose(0, 1).contiguous().transpose(0, 1)), "same strides"),
])
def test_quantised_caches_that_do_not_fit_are_refused(spoil, what):
    kc, vc, ke, ve = spoil(_cache(True))
    x = torch.zeros(3, H, D, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match=what):
        ops.cache_write(x, x, kc, vc, SLOTS, ke, ve)
    with pytest.raises(RuntimeError, match=what):
        ops.cache_read(kc, vc, SLOTS, ke, ve, dtype=torch.bfloat16)


def _attend(**change):
    kc, vc, _, _ = _cache()
    a = dict(query=torch.zeros(3, 4, D, dtype=torch.float16), key_cache=kc, value_cache=vc, page_table=torch.zeros(3, 2, dtype=torch.int32),
             lengths=torch.ones(3, dtype=torch.int32)) | change
    return ops.paged_attention(**a)


Q = torch.zeros(3, 4, D, dtype=torch.float16)


@pytest.mark.parametrize("change,what", [
    (dict(), "CUDA"), (dict(lengths=torch.ones(3, dtype=torch.int64)), "lengths"), (dict(lengths=torch.ones(2, dtype=torch.int32)), "lengths"),
    (dict(query_starts=torch.ones(3, dtype=torch.int32)), "query_starts"), (dict(query_starts=torch.ones(8, dtype=torch.int32)[::2]), "query_starts"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), "page_table"), (dict(page_table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), "page_table"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32)), "query_starts is needed"),
    (dict(window=0), "window"), (dict(window=-3), "window"), (dict(window=3, causal=False), "window"), (dict(query=Q[:, :3]), "do not go with"),
    (dict(query=Q[:, :0]), "do not go with"), (dict(query=Q[..., :32]), "do not go with"), (dict(query=Q.bfloat16()), "the cache holds"),
    (dict(query=Q[0]), "query must be"), (dict(query=Q.transpose(1, 2)), "query must be"), (dict(out=Q.float()), "out must"), (dict(out=Q[:2]), "out must"),
])
def test_attention_refuses_what_does_not_fit(change, what):
    with pytest.raises(RuntimeError, match=what):
        _attend(**change)


def test_what_is_no_tensor_is_a_type_error():
    with pytest.raises(TypeError, match="lengths"):
        _attend(lengths=[1, 1, 1])
    with pytest.raises(TypeError, match="key_exponents"):
        _attend(key_exponents=3)


@pytest.mark.parametrize("change,what", [
    (dict(), "CUDA"), (dict(positions=torch.zeros(2, dtype=torch.int32)), "positions"), (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(key=Q.view(3, 256)), "key"), (dict(key=Q.view(3, 256)[:2].bfloat16()), "key must have"), (dict(head_size=48), "query must be"),
    (dict(head_size=0), "query must be"), (dict(query=Q[:2, :, ::2].flatten(1)[:, ::2]), "query must be"),
    (dict(cos_sin_cache=torch.zeros(8, 64, dtype=torch.float64)), "cos_sin_cache"), (dict(cos_sin_cache=torch.zeros(8, 128)[:, ::2]), "cos_sin_cache"),
    (dict(query_weight=torch.zeros(32, dtype=torch.float16)), "weight"), (dict(key_weight=torch.zeros(64)), "weight"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(query_out=Q.view(3, 256)), "query_out"), (dict(key_out=Q.view(3, 256)), "key_out"),
])
def test_norm_and_rotation_refuse_what_does_not_fit(change, what):
    a = dict(positions=torch.zeros(2, dtype=torch.int64), query=Q[:2].flatten(1).clone(), key=Q[:2].flatten(1).clone(), head_size=64,
             cos_sin_cache=torch.zeros(8, 64), is_neox=True) | change
    with pytest.raises(RuntimeError, match=what):
        capi.qk_norm_rotary_embedding(**a)


def test_a_missing_binding_fails_loudly(monkeypatch):
    import sys

    import triteia_b200

    monkeypatch.setitem(sys.modules, "triteia_b200._binding", None)      # what an import that finds nothing leaves
    monkeypatch.delattr(triteia_b200, "_binding", raising=False)
    with pytest.raises(ImportError, match="no CPU"):
        _lib.load_binding()


def test_a_window_that_leaves_32_bits_is_refused():
    """Positions run from -num_tokens to the table's width, and a window is subtracted from them."""
    assert _attention(table_width=1 << 25, page_size=63, num_tokens=1 << 29, window=5) == 1


def test_what_ctypes_binds_does_without_the_extension_module():
    """It is built for one Python and one torch: the package imports without it, and only the operators that it binds say that it
    is missing."""
    import subprocess
    import sys

    code = """
import sys
sys.modules["triteia_b200._binding"] = None
import torch
from triteia_b200 import capi, nn, ops, triteia_cuda
qweight, q, s, meta = ops.gen_sparse_quant4_NT(256, 128, device="cpu")
try:
    ops.matmul_4bit_2_4(q, torch.randn(4, 128).half(), meta, s)
except RuntimeError as e:
    assert "CUDA" in str(e)
x, slots = torch.zeros(3, 2, 64).half(), torch.zeros(3, dtype=torch.int64)
for call in (lambda: ops.cache_write(x, x, x, x, slots), lambda: ops.cache_read(x, x, slots), lambda: ops.paged_attention(x, x, x, slots, slots),
             lambda: capi.qk_norm_rotary_embedding(slots, x, x, 64, x, True)):
    try:
        call()
    except ImportError as e:
        assert "triteia_b200.build" in str(e)
    else:
        raise AssertionError("no error")
print("fine")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert res.returncode == 0 and "fine" in res.stdout, res.stderr


def test_an_extension_module_for_another_torch_is_built_again(monkeypatch, tmp_path):
    from triteia_b200 import build

    assert build.binding_fits() and _lib.load_binding().built_for == build.binding_tag()
    made = []

    def compiled(cmd, **kw):
        made.append(cmd)
        return type("Result", (), dict(returncode=0, stdout="", stderr=""))()

    monkeypatch.setattr(build.subprocess, "run", compiled)
    build.build_binding()
    assert not made                                    # it is there, newer than its sources, and fits
    monkeypatch.setattr(build, "binding_tag", lambda: "triteia_b200 binding, torch 99.0, cpython-399")
    build.build_binding()
    assert len(made) == 1 and any("torch 99.0" in x for x in made[0])
    with pytest.raises(ImportError, match="torch 99.0.*triteia_b200.build"):
        _lib.load_binding()
    assert not build.binding_fits(str(tmp_path / "none.so"))


def test_workspace_only_for_the_calls_that_use_one():
    def needs(tokens, seqs, page, width, head_stride=64, single=0):
        return _lib.lib.trb_paged_attention_cache_workspace_bytes(tokens, seqs, 8, 2, 64, page, 100, width, page * 128, 128, head_stride, single, 0, 0)

    assert needs(700, 3, 16, 200) == 0                 # tensor memory
    for args in (dict(page=24), dict(page=16, head_stride=0)):
        assert needs(700, 3, width=200, **args) == _lib.lib.trb_paged_attention_workspace_bytes(700, 3, 8, 2, 64, args["page"], 200, 0, 0, 0)
    for tokens, single in ((3, 1), (3, 0)):
        assert needs(tokens, 3, 16, 200, single=single) == _lib.lib.trb_paged_attention_workspace_bytes(tokens, 3, 8, 2, 64, 16, 200, single, 0, 0)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1e300, -3e38])
def test_a_scale_that_is_no_finite_number_is_refused(scale):
    kc, vc, _, _ = ops.new_cache(PAGES, P, H, D, device="cpu")
    x = torch.zeros(3, H, D, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="scale"):
        ops.paged_attention(x, kc, vc, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32), scale=scale)
    if abs(scale) < 1e39 or scale != scale or abs(scale) == float("inf"):
        assert _attention(scale=scale) == 3
