"""The paged cache's argument checks, on the CPU: the C structs' layout, every refusal of the C ABI (they come
before any launch) and of the Python front end."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from gemma4_posttrain_jax_amd import _lib, kernels
from gemma4_posttrain_jax_amd.kvcache import PagedLayerCache, new_paged_layer

HEADER = Path(__file__).resolve().parents[1] / "include" / "g4_rollout.h"


def test_paged_structs_match_the_compiled_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for st in (_lib.G4PagedCache, _lib.G4PagedAppendArgs, _lib.G4PagedDecodeArgs, _lib.G4PagedReadArgs):
        lines.append(f'printf("{st.__name__} size %zu\\n", sizeof({st.__name__}));')
        lines += [f'printf("{st.__name__} {f} %zu\\n", offsetof({st.__name__}, {f}));' for f, _ in st._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line in filter(None, out):
        name, field, value = line.split()
        st = getattr(_lib, name)
        assert (ctypes.sizeof(st) if field == "size" else getattr(st, field).offset) == int(value), line


def _cache(**kw):
    base = dict(format=_lib.G4_PAGES_E4M3, num_pages=8, kv_heads=2, head_dim=256, page_size=64, key=1 << 12,
                value=1 << 12, key_scale=1 << 12, value_scale=1 << 12)
    base.update(kw)
    return _lib.G4PagedCache(**base)


def _append(cache=None, **kw):
    base = dict(cache=_cache(**(cache or {})), batch=2, seq=3, group=4, flags=0, eps=1e-6, keep=0, max_pages=4,
                table_stride=4, page_table=1 << 12, write_pos=1 << 12, k=1 << 12, v=1 << 12, q=None,
                in_row_stride=2048, q_norm_weight=None, k_norm_weight=None, rope_cos=None, rope_sin=None, q_out=None)
    base.update(kw)
    return _lib.G4PagedAppendArgs(**base)


def _decode(cache=None, **kw):
    base = dict(cache=_cache(**(cache or {})), batch=2, group=4, window=0, max_pages=4, table_stride=4,
                page_table=1 << 12, lengths=1 << 12, q=1 << 12, out=1 << 12, workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.G4PagedDecodeArgs(**base)


def _read(cache=None, **kw):
    base = dict(cache=_cache(**(cache or {})), batch=2, start=0, count=10, max_pages=4, table_stride=4,
                page_table=1 << 12, lengths=1 << 12, k_out=1 << 12, v_out=1 << 12)
    base.update(kw)
    return _lib.G4PagedReadArgs(**base)


CALLS = [("g4_paged_append", _append), ("g4_paged_decode_attention", _decode), ("g4_paged_read", _read)]


def _refused(name, args, match):
    rc = getattr(_lib.lib(), name)(ctypes.byref(args), None)
    assert rc in (_lib.G4_ERR_INVALID, _lib.G4_ERR_UNSUPPORTED), rc
    text = _lib.lib().g4_last_error().decode()
    assert re.search(match, text) and name in text, text


@pytest.mark.parametrize("name,make", CALLS)
@pytest.mark.parametrize("override,match", [
    (dict(format=2), "format"), (dict(num_pages=0), "num_pages"), (dict(kv_heads=0), "kv_heads"),
    (dict(head_dim=32), "head_dim"), (dict(head_dim=192), "head_dim"), (dict(page_size=16), "page_size"),
    (dict(page_size=96), "page_size"), (dict(page_size=2048), "page_size"), (dict(key=None), "NULL"),
    (dict(value=(1 << 12) + 8), "aligned"), (dict(key_scale=None), "key_scale"),
    (dict(value_scale=(1 << 12) + 4), "aligned"),
])
def test_abi_refuses_bad_pages(name, make, override, match):
    _refused(name, make(override), match)


@pytest.mark.parametrize("name,make", CALLS)
@pytest.mark.parametrize("override,match", [
    (dict(batch=0), "batch"), (dict(page_table=None), "page table"), (dict(max_pages=0), "page table"),
    (dict(table_stride=3), "page table"), (dict(max_pages=1 << 26, table_stride=1 << 26), "positions"),
])
def test_abi_refuses_bad_tables(name, make, override, match):
    _refused(name, make(**override), match)


@pytest.mark.parametrize("name,make,override,match", [
    ("g4_paged_append", _append, dict(seq=0), "seq"),
    ("g4_paged_append", _append, dict(keep=-1), "keep"),
    ("g4_paged_append", _append, dict(batch=1 << 20, seq=1 << 20), "tokens"),
    ("g4_paged_append", _append, dict(batch=1 << 20, seq=1 << 10), "tokens"),  # a grid of 2^32 threads or more
    ("g4_paged_append", _append, dict(batch=1 << 24, seq=1, in_row_stride=512), "tokens"),
    ("g4_paged_append", _append, dict(k=None), "NULL"),
    ("g4_paged_append", _append, dict(write_pos=None), "NULL"),
    ("g4_paged_append", _append, dict(q=1 << 12), "q_out"),
    ("g4_paged_append", _append, dict(q=1 << 12, q_out=1 << 12, group=0), "group"),
    ("g4_paged_append", _append, dict(q=1 << 12, q_out=(1 << 12) + 4), "q_out"),
    ("g4_paged_append", _append, dict(in_row_stride=500), "in_row_stride"),
    ("g4_paged_append", _append, dict(q=1 << 12, q_out=1 << 12, in_row_stride=2047), "in_row_stride"),
    ("g4_paged_append", _append, dict(q=1 << 12, q_out=1 << 12, group=1 << 20, in_row_stride=1 << 40), "heads"),
    ("g4_paged_append", _append, dict(flags=_lib.G4_APPEND_ROPE_K), "RoPE"),
    ("g4_paged_append", _append, dict(flags=_lib.G4_APPEND_NORM_K), "k_norm_weight"),
    ("g4_paged_append", _append, dict(q=1 << 12, q_out=1 << 12, flags=_lib.G4_APPEND_NORM_Q), "q_norm_weight"),
    ("g4_paged_decode_attention", _decode, dict(group=0), "group"),
    ("g4_paged_decode_attention", _decode, dict(group=17), "group"),
    ("g4_paged_decode_attention", _decode, dict(window=-1), "window"),
    ("g4_paged_decode_attention", _decode, dict(batch=1 << 24), "batch"),
    ("g4_paged_decode_attention", _decode, dict(batch=1 << 16, max_pages=1 << 18, table_stride=1 << 18), "positions"),
    ("g4_paged_decode_attention", _decode, dict(lengths=None), "NULL"),
    ("g4_paged_decode_attention", _decode, dict(out=None), "NULL"),
    ("g4_paged_decode_attention", _decode, dict(q=(1 << 12) + 2), "aligned"),
    ("g4_paged_read", _read, dict(start=-1), "start"),
    ("g4_paged_read", _read, dict(count=0), "count"),
    ("g4_paged_read", _read, dict(start=2**31 - 1000, count=100), "count"),
    ("g4_paged_read", _read, dict(batch=1 << 20, count=1 << 20), "positions"),
    ("g4_paged_read", _read, dict(batch=1 << 18, count=1 << 12), "positions"),
    ("g4_paged_decode_attention", _decode, dict(batch=0x3fffff), "batch"),
    ("g4_paged_read", _read, dict(k_out=None), "NULL"),
    ("g4_paged_read", _read, dict(v_out=(1 << 12) + 8), "aligned"),
])
def test_abi_refuses_bad_calls(name, make, override, match):
    _refused(name, make(**override), match)


def test_abi_refuses_null_args():
    for name, _ in CALLS:
        assert getattr(_lib.lib(), name)(None, None) == _lib.G4_ERR_INVALID
    assert _lib.lib().g4_paged_decode_workspace_size(None) == 0


def test_abi_checks_the_attention_workspace():
    """Rows that one workgroup takes need none; longer ones a fixed number of slots, whatever the lengths."""

    L = _lib.lib()
    assert L.g4_paged_decode_workspace_size(ctypes.byref(_decode())) == 0
    long = dict(max_pages=1000, table_stride=1000)
    need = L.g4_paged_decode_workspace_size(ctypes.byref(_decode(**long)))
    assert 0 < need == L.g4_paged_decode_workspace_size(ctypes.byref(_decode(max_pages=5000, table_stride=5000)))
    assert L.g4_paged_decode_workspace_size(ctypes.byref(_decode(**long, window=512))) == 0
    for ws, size in ((None, need), (1 << 12, need - 1), ((1 << 12) + 4, need)):
        a = _decode(**long, workspace=ws, workspace_bytes=size)
        assert L.g4_paged_decode_attention(ctypes.byref(a), None) == _lib.G4_ERR_WORKSPACE
        assert re.search("workspace", L.g4_last_error().decode())


def test_new_paged_layer():
    for e4m3 in (False, True):
        layer = new_paged_layer(3, 2, 128, 64, e4m3=e4m3, device="cpu")
        assert (layer.num_pages, layer.kv_heads, layer.page_size, layer.head_dim, layer.e4m3) == (3, 2, 64, 128, e4m3)
        assert layer.key.numel() == layer.value.numel() == 3 * 2 * 64 * 128
        assert (layer.key_scale is None) == (not e4m3)
    for bad in (dict(num_pages=0), dict(kv_heads=0), dict(head_dim=96), dict(page_size=48)):
        with pytest.raises(ValueError):
            new_paged_layer(**{**dict(num_pages=1, kv_heads=1, head_dim=64, page_size=32, device="cpu"), **bad})


def _layer(e4m3=False):
    return new_paged_layer(4, 2, 64, 32, e4m3=e4m3, device="cpu")


def _table(B=3, M=2):
    return torch.zeros((B, M), dtype=torch.int32), torch.ones(B, dtype=torch.int32)


def test_front_end_refuses_bad_operands():
    table, n = _table()
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    layer, k = _layer(), bf(3, 5, 2, 64)
    append = lambda layer=layer, k=k, v=k, **kw: kernels.paged_append(  # noqa: E731
        layer, k, v, **{**dict(page_table=table, write_pos=n), **kw})
    attend = lambda layer=layer, q=bf(3, 2, 4, 64), **kw: kernels.paged_decode_attention(  # noqa: E731
        layer, q, **{**dict(page_table=table, lengths=n), **kw})
    read = lambda layer=layer, **kw: kernels.paged_read(  # noqa: E731
        layer, **{**dict(page_table=table, lengths=n, start=0, count=4), **kw})
    for call in (append, attend, read):
        with pytest.raises(ValueError, match="page_table"):
            call(page_table=table.long())
        with pytest.raises(ValueError, match="page_table"):
            call(page_table=table.t())
        with pytest.raises(ValueError, match="page_table"):
            call(page_table=table[:, :0])
        with pytest.raises(ValueError, match="device tensors"):
            call()
        with pytest.raises(TypeError, match="pages of"):
            call(layer=PagedLayerCache(layer.key.float(), layer.value.float()))
        with pytest.raises(ValueError, match="do not match"):
            call(layer=PagedLayerCache(layer.key[:1], layer.value))
        with pytest.raises(ValueError, match="no scales"):
            call(layer=PagedLayerCache(layer.key, layer.value, n, n))
        e = _layer(True)
        with pytest.raises(ValueError, match="scales"):
            call(layer=PagedLayerCache(e.key, e.value))
        with pytest.raises(ValueError, match="scales"):
            call(layer=PagedLayerCache(e.key, e.value, e.key_scale.view(torch.uint8), e.value_scale))
    for call, name in ((append, "write_pos"), (attend, "lengths"), (read, "lengths")):
        with pytest.raises(ValueError, match=name):
            call(**{name: n.long()})
        with pytest.raises(ValueError, match=name):
            call(**{name: n[:2]})
    with pytest.raises(ValueError, match="batch"):
        append(k=k[:2], v=k[:2])
    with pytest.raises(TypeError, match="bfloat16"):
        append(k=k.float(), v=k.float())
    with pytest.raises(ValueError, match="pages of"):
        append(k=bf(3, 5, 1, 64), v=bf(3, 5, 1, 64))
    with pytest.raises(ValueError, match="v: "):
        append(v=bf(3, 5, 2, 128)[..., ::2])
    with pytest.raises(ValueError, match="keep"):
        append(keep=-1)
    with pytest.raises(ValueError, match="q_out"):
        append(k=bf(3, 5, 2 * 64 * 3)[..., :128].view(3, 5, 2, 64), v=bf(3, 5, 2 * 64 * 3)[..., :128].view(3, 5, 2, 64),
               q=bf(3, 5, 2 * 64 * 3)[..., :128].view(3, 5, 2, 1, 64))
    with pytest.raises(ValueError, match="k_norm_weight"):
        append(flags=_lib.G4_APPEND_NORM_K, k_norm_weight=bf(32))
    with pytest.raises(ValueError, match="rope"):
        append(flags=_lib.G4_APPEND_ROPE_K, rope_cos=torch.zeros(3, 5, 64), rope_sin=torch.zeros(3, 4, 64))
    with pytest.raises(ValueError, match="q must"):
        attend(q=bf(3, 2, 64, 4).transpose(2, 3))
    with pytest.raises(ValueError, match="batch"):
        attend(q=bf(2, 2, 4, 64))
    with pytest.raises(ValueError, match="window"):
        attend(window=-1)
    with pytest.raises(ValueError, match="out must"):
        attend(out=bf(3, 2, 5, 64))
    with pytest.raises(ValueError, match="start"):
        read(start=-1)
    with pytest.raises(ValueError, match="count"):
        read(count=0)


def test_init_paged_kv_cache():
    import hf_util as H
    from gemma4_posttrain_jax_amd import config as C
    from gemma4_posttrain_jax_amd.kvcache import PagedSpec, init_paged_kv_cache

    cfg = C.config_from_hf(dict(H.CFG1, sliding_window=40))
    cache = init_paged_kv_cache(cfg, 3, 200, PagedSpec(32), device="cpu")
    assert cache.batch == 3 and cache.capacity == 224 and cache.length == 0
    assert tuple(cache.page_table.shape) == tuple(cache.window_table.shape) == (3, 7)
    cycle = 3  # 40 positions touch 2 or 3 pages of 32
    for i, layer in enumerate(cache.layers):
        sliding = cfg.layer_types[i] == C.SLIDING
        table = cache.window_table if sliding else cache.page_table
        assert layer.num_pages == 3 * (cycle if sliding else 7)
        assert int(table.min()) == 0 and int(table.max()) == layer.num_pages - 1
        for b in range(3):
            assert len(set(table[b].tolist())) == (cycle if sliding else 7)
            for j in range(7 - cycle):  # no page twice within a window
                assert len(set(table[b, j: j + cycle].tolist())) == cycle
    for bad in (dict(batch_size=0), dict(capacity=0), dict(spec=PagedSpec(40))):
        with pytest.raises(ValueError):
            init_paged_kv_cache(cfg, **{**dict(batch_size=1, capacity=10, device="cpu"), **bad})
