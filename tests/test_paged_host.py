"""CPU-only tests of the paged-cache group's host side: the C ABI and its refusals, the facade, the schemas and
fake kernels, the frequencies.  No kernel is launched."""
import ctypes
import math
import os
import re

import pytest
import torch

from custom_ops_b200 import CustomOpsError, FAOps, PagedOps, RecsysOps, _cabi_paged as abi, build, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "fa_paged_sm100.h")
P = 4096                                   # a 16-byte aligned address that is never touched


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build_paged_binding()


def test_library_exports_every_declared_symbol():
    declared = set(re.findall(r"^(?:int|const char\*)\s+(fa_\w+)\s*\(", open(HEADER).read(), flags=re.M))
    assert declared == set(abi.EXPORTS)
    lib = abi.load()
    for name in declared:
        assert getattr(lib, name) is not None
    assert lib.fa_paged_sm100_strerror(0) == b"ok" and lib.fa_paged_sm100_strerror(-99) == b"unknown error"
    for code in range(-11, 0):
        assert lib.fa_paged_sm100_strerror(code) not in (b"ok", b"unknown error")
    assert lib.fa_paged_sm100_launch_count(None) == -1
    assert abi.launch_count() >= 0


def test_struct_sizes_match_header_layout():
    assert ctypes.sizeof(abi.PagedCacheView) == 2 * 8 + 6 * 8 + 4 * 4
    assert ctypes.sizeof(abi.RotarySpec) == 2 * 8 + 6 * 4
    assert ctypes.sizeof(abi.ExtendArgs) == 8 + 2 * 8 + 9 * 8 + 4 * 4 + 8
    assert ctypes.sizeof(abi.ShrinkArgs) == 8 + 2 * 8 + 4 * 8 + 4 * 4
    assert ctypes.sizeof(abi.RotaryArgs) == 8 + 4 * 8 + 7 * 8 + 40 + 6 * 4
    assert ctypes.sizeof(abi.AppendArgs) == 8 + 5 * 8 + 6 * 8 + 80 + 40 + 8 + 4 * 4
    assert ctypes.sizeof(abi.AttentionArgs) == 8 + 6 * 8 + 3 * 8 + 80 + 4 * 4 + 2 * 4 + 2 * 4


def fill(cls, **kw):
    a = cls()
    a.struct_size = ctypes.sizeof(cls)
    for path, value in kw.items():
        at = a
        *outer, last = path.split("__")
        for name in outer:
            at = getattr(at, name)
        setattr(at, last, value)
    return a


def cache(**kw):
    base = dict(cache__k=P, cache__v=P, cache__num_pages=8, cache__heads_k=2, cache__page_size=16, cache__head_dim=64)
    for t in "kv":
        base.update({f"cache__{t}_page_stride": 2048, f"cache__{t}_head_stride": 1024, f"cache__{t}_row_stride": 64})
    base.update(kw)
    return base


def attention(**kw):
    base = dict(q=P, out=P, block_table=P, lens=P, q_batch_stride=256, q_head_stride=64, table_stride=4, batch=2, heads=4,
                table_width=4, scale=0.125, dtype=abi.BF16)
    base.update(cache())
    base.update(kw)
    return fill(abi.AttentionArgs, **base)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -11), (dict(dtype=7), -2), (dict(device=-1), -3), (dict(device=64), -3),
    (dict(batch=-1), -3), (dict(heads=3), -3), (dict(table_width=-1), -3), (dict(table_stride=-4), -3),
    (dict(cache__heads_k=0), -3), (dict(cache__page_size=0), -3), (dict(cache__num_pages=-1), -3),
    (dict(cache__head_dim=96), -4), (dict(cache__head_dim=256), -4), (dict(cache__k=None), -1), (dict(cache__v=None), -1),
    (dict(cache__k=P + 8), -5), (dict(q=P + 2), -5), (dict(out=P + 4), -5), (dict(q_head_stride=68), -5),
    (dict(cache__v_row_stride=65), -5), (dict(cache__k_page_stride=-8), -5),
    (dict(window=-1), -10), (dict(softcap=-1.0), -10), (dict(softcap=float("nan")), -10), (dict(scale=float("inf")), -10),
    (dict(scale=-0.5), -10), (dict(scale=3e38), -10), (dict(softcap=1e-45), -10), (dict(table_width=1 << 28), -3), (dict(batch=1 << 20, heads=1 << 12), -3),
])
def test_attention_refusals(kw, code):
    with pytest.raises(abi.PagedError) as e:
        abi.workspace_bytes(attention(**kw))
    assert e.value.code == code
    assert abi.load().fa_paged_attention_sm100(ctypes.byref(attention(**kw)), None, 0, None) == code


def test_attention_of_nothing_needs_nothing():
    assert abi.workspace_bytes(attention(batch=0)) == 0
    assert abi.workspace_bytes(attention(heads=0)) == 0
    assert abi.load().fa_paged_attention_sm100(ctypes.byref(attention(batch=0)), None, 0, None) == 0
    assert abi.load().fa_paged_attention_sm100(None, None, 0, None) == -1
    assert abi.load().fa_paged_attention_sm100_workspace_bytes(ctypes.byref(attention()), None) == -1


def rotary_args(**kw):
    base = dict(q=P, k=P, q_out=P, k_out=P, rotary__freqs=P, rotary__positions=P, rotary__rot_dim=64, rotary__mscale=1.0,
                batch=1, heads=4, heads_k=2, seqlen=8, head_dim=64, dtype=abi.BF16, q_row_stride=64, q_head_stride=512)
    base.update(kw)
    return fill(abi.RotaryArgs, **base)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=0), -11), (dict(dtype=2), -2), (dict(device=99), -3), (dict(batch=-1), -3), (dict(batch=65536), -3),
    (dict(seqlen=-1), -3), (dict(heads=-2), -3), (dict(heads_k=-2), -3), (dict(position_batch_stride=-1), -3),
    (dict(head_dim=80), -4), (dict(q=P + 8), -5), (dict(k_out=P + 8), -5), (dict(q_row_stride=60), -5),
    (dict(k_batch_stride=-64), -5), (dict(rotary__freqs=None), -1), (dict(rotary__positions=None), -1),
    (dict(rotary__rot_dim=63), -9), (dict(rotary__rot_dim=0), -9), (dict(rotary__rot_dim=66), -9),
    (dict(rotary__mscale=float("nan")), -9), (dict(q=None), -1), (dict(k_out=None), -1),
])
def test_rotary_refusals(kw, code):
    assert abi.load().fa_rotary_sm100(ctypes.byref(rotary_args(**kw)), None) == code


def append_args(**kw):
    base = dict(q=P, k=P, v=P, q_out=P, slots=P, rotary__freqs=P, rotary__positions=P, rotary__rot_dim=64,
                rotary__mscale=1.0, num_tokens=4, heads=4, dtype=abi.BF16, k_token_stride=128, k_head_stride=64)
    base.update(cache())
    base.update(kw)
    return fill(abi.AppendArgs, **base)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=1), -11), (dict(dtype=-1), -2), (dict(device=-2), -3), (dict(num_tokens=-1), -3), (dict(heads=-1), -3),
    (dict(num_tokens=1 << 31), -3), (dict(cache__page_size=0), -3), (dict(cache__head_dim=32), -4),
    (dict(cache__v=P + 8), -5), (dict(v=P + 2), -5), (dict(k_token_stride=1), -5), (dict(rotary__rot_dim=65), -9),
    (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1), (dict(q=None), -1), (dict(q_out=None), -1),
    (dict(rotary__positions=None), -1),
])
def test_append_refusals(kw, code):
    assert abi.load().fa_paged_append_sm100(ctypes.byref(append_args(**kw)), None) == code


def test_rotary_and_append_of_nothing():
    lib = abi.load()
    for kw in (dict(batch=0), dict(seqlen=0), dict(heads=0, heads_k=0)):
        assert lib.fa_rotary_sm100(ctypes.byref(rotary_args(**kw)), None) == 0
    assert lib.fa_paged_append_sm100(ctypes.byref(append_args(num_tokens=0)), None) == 0
    assert lib.fa_rotary_sm100(None, None) == lib.fa_paged_append_sm100(None, None) == -1


def table_args(cls, **kw):
    base = dict(block_table=P, table_stride=4, lens=P, free_pages=P, free_head=P, batch=3, table_width=4, page_size=16,
                num_free_pages=9)
    base.update(dict(new_lens=P, lens_out=P, head_out=P, slots=P, positions=P, cu=P, num_tokens=5)
                if cls is abi.ExtendArgs else dict(keep_lens=P))
    base.update(kw)
    return fill(cls, **base)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=2), -11), (dict(device=-1), -3), (dict(batch=-1), -3), (dict(batch=16385), -3), (dict(table_width=-1), -3),
    (dict(page_size=0), -3), (dict(num_free_pages=-1), -3), (dict(table_width=1 << 30), -3), (dict(block_table=None), -1),
    (dict(lens=None), -1), (dict(free_pages=None), -1), (dict(free_head=None), -1),
])
def test_table_refusals(kw, code):
    lib = abi.load()
    assert lib.fa_paged_extend_sm100(ctypes.byref(table_args(abi.ExtendArgs, **kw)), None) == code
    assert lib.fa_paged_shrink_sm100(ctypes.byref(table_args(abi.ShrinkArgs, **kw)), None) == code


def test_more_table_refusals():
    lib = abi.load()
    for kw, code in ((dict(num_tokens=-1), -3), (dict(cu=None), -1), (dict(new_lens=None), -1), (dict(lens_out=None), -1),
                     (dict(head_out=None), -1), (dict(slots=None), -1), (dict(positions=None), -1)):
        assert lib.fa_paged_extend_sm100(ctypes.byref(table_args(abi.ExtendArgs, **kw)), None) == code
    assert lib.fa_paged_shrink_sm100(ctypes.byref(table_args(abi.ShrinkArgs, keep_lens=None)), None) == -1
    assert lib.fa_paged_shrink_sm100(ctypes.byref(table_args(abi.ShrinkArgs, batch=0, lens=None)), None) == 0
    assert lib.fa_paged_extend_sm100(None, None) == lib.fa_paged_shrink_sm100(None, None) == -1


def test_without_a_gpu_every_call_fails_loudly():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib = abi.load()
    for call, args in ((lib.fa_paged_extend_sm100, table_args(abi.ExtendArgs)),
                       (lib.fa_paged_shrink_sm100, table_args(abi.ShrinkArgs)),
                       (lib.fa_rotary_sm100, rotary_args()), (lib.fa_paged_append_sm100, append_args())):
        assert call(ctypes.byref(args), None) in (-7, -8)
    with pytest.raises(abi.PagedError) as e:
        abi.workspace_bytes(attention())
    assert e.value.code in (-7, -8)


# ------------------------------------------------------------------ loader / facade
def test_group_is_listed_once_it_is_asked_for():
    fresh = RecsysOps()
    assert fresh.groups == {"fa": "not_loaded"}
    assert callable(fresh.paged_attention)                          # looking at the method loads nothing
    assert fresh.groups == {"fa": "not_loaded"}
    fresh.ensure_loaded("paged")
    assert fresh.groups == {"fa": "not_loaded", "paged": "loaded"}, fresh.load_error("paged")
    assert fresh.is_available("paged") and fresh.load_error("paged") is None
    with pytest.raises(ValueError, match="paged"):
        fresh.ensure_loaded("moe")
    with pytest.raises(AttributeError, match="paged_attention"):
        fresh.no_such_op
    with pytest.raises(CustomOpsError):
        fresh.rotary(None, None, None, None, backend="tilelang")


def test_schemas_and_fake_kernels():
    ops = RecsysOps().ensure_loaded("paged")
    assert set(PagedOps.required_ops) == set(PagedOps.op_schemas) == set(PagedOps.fake_ops)
    meta = dict(device="meta")
    q = torch.empty(3, 8, 64, dtype=torch.bfloat16, **meta)
    kv = torch.empty(3, 2, 64, dtype=torch.bfloat16, **meta)
    kc = torch.empty(5, 2, 16, 64, dtype=torch.bfloat16, **meta)
    i32 = torch.empty(3, dtype=torch.int32, **meta)
    table = torch.empty(3, 4, dtype=torch.int32, **meta)
    freqs = torch.empty(32, dtype=torch.float64, **meta)
    out, lse = ops.paged_attention_lse(q, kc, kc, table, i32)
    assert out.shape == q.shape == ops.paged_attention(q, kc, kc, table, i32).shape
    assert lse.shape == (3, 8) and lse.dtype == torch.float32
    assert ops.rotary_append(q, kv, kv, i32, i32, kc, kc, freqs).shape == q.shape
    assert ops.paged_append(kv, kv, i32, kc, kc) is None
    a, b = ops.rotary(torch.empty(1, 9, 8, 64, dtype=torch.bfloat16, **meta).transpose(1, 2),
                      torch.empty(1, 2, 9, 64, dtype=torch.bfloat16, **meta), torch.empty(9, dtype=torch.int32, **meta), freqs)
    assert a.shape == (1, 8, 9, 64) and a.is_contiguous() and b.shape == (1, 2, 9, 64)
    lens, head, slots, positions, cu = ops.paged_extend(table, i32, i32, i32, i32[:1], 16, 7)
    assert lens.shape == (3,) and head.shape == (1,) and slots.shape == positions.shape == (7,) and cu.shape == (4,)
    assert slots.dtype == torch.int64 and positions.dtype == cu.dtype == torch.int32
    assert len(ops.paged_extend_(table, i32, i32, i32, i32[:1], 16, 7)) == 3
    assert ops.paged_shrink_(table, i32, i32, i32, i32[:1], 16) is None


def test_cpu_tensors_are_refused():
    ops = RecsysOps()
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    kc = torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.paged_attention(x, kc, kc, i.view(1, 1), i), lambda: ops.paged_append(x, x, i, kc, kc),
                 lambda: ops.paged_extend(i.view(1, 1), i, i, i, i, 8, 1),
                 lambda: ops.rotary(kc, kc, torch.zeros(8, dtype=torch.int32), torch.zeros(4, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="only supported on CUDA"):
            call()


def test_export_and_strict_load_of_the_group(tmp_path):
    path = PagedOps().export(str(tmp_path))
    assert sorted(os.listdir(tmp_path)) == ["libfa_paged_sm100.so", "recsys_paged_kernel.so", "recsys_paged_kernel.so.json"]
    from custom_ops_b200 import deploy
    assert deploy.check_precompiled(PagedOps(), path)["schemas"].keys() == PagedOps.op_schemas.keys()
    with pytest.raises(CustomOpsError):
        deploy.check_precompiled(FAOps(), path)


def test_sources_read_nothing_through_the_read_only_path_and_spill_nothing():
    code = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "custom_ops_b200", "csrc", "fa_paged_sm100.cu")).read())
    assert not re.findall(r"__ldg\b|__restrict__|ld\.global\.nc", code)
    build.build_paged_cabi()
    assert build.spilled_bytes(build.PAGED_CABI_SO) == 0


# ------------------------------------------------------------------ frequencies
def test_rotary_frequencies():
    f, m = rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0
    assert all(abs(f[i].item() - 10000.0 ** (-2 * i / 64)) < 1e-16 for i in range(32))
    g, m = rotary_frequencies(64, 10000.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(g, f / 4) and m == 1.0
    g, m = rotary_frequencies(64, 10000.0, scaling="base", factor=4.0, device="cpu")
    assert g[0] == f[0] and abs(g[-1].item() * 4 / f[-1].item() - 1) < 1e-12 and m == 1.0
    g, m = rotary_frequencies(64, 10000.0, scaling="by_parts", factor=4.0, original_length=4096, device="cpu")
    assert abs(m - (0.1 * math.log(4.0) + 1)) < 1e-15
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.7], f[turns < 0.7] / 4, rtol=1e-12)
    assert ((g <= f) & (g >= f / 4 * (1 - 1e-12))).all() and (g[1:] < g[:-1]).all()
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.5),
                dict(rot_dim=8, scaling="other"), dict(rot_dim=2, scaling="base"), dict(rot_dim=8, scaling="by_parts"),
                dict(rot_dim=8, scaling="by_parts", original_length=10, slow=5.0, fast=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **bad)
