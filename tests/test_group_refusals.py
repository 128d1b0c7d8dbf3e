"""What packed attention, the page pool and the drafts' verification refuse, on the CPU: the C structs' layout, the C
ABI's checks (they come before any launch) and the Python front end's."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from gemma4_posttrain_jax_amd import _lib, kernels
from gemma4_posttrain_jax_amd.kvcache import key_shape, new_paged_layer, page_counts

HEADER = Path(__file__).resolve().parents[1] / "include" / "g4_rollout.h"
AT = 1 << 12  # an address that no check before a launch reads


def test_structs_match_the_compiled_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for st in (_lib.G4PackedPrefillArgs, _lib.G4PageTable, _lib.G4PagedReserveArgs, _lib.G4PagedForkArgs, _lib.G4PagedFreeArgs,
               _lib.G4PagedCompactArgs, _lib.G4VerifyArgs):
        lines.append(f'printf("{st.__name__} size %zu\\n", sizeof({st.__name__}));')
        lines += [f'printf("{st.__name__} {f} %zu\\n", offsetof({st.__name__}, {f}));' for f, _ in st._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line in filter(None, out):
        name, field, value = line.split()
        st = getattr(_lib, name)
        assert (ctypes.sizeof(st) if field == "size" else getattr(st, field).offset) == int(value), line


def _refused(name, args, match, codes=(_lib.G4_ERR_INVALID, _lib.G4_ERR_UNSUPPORTED)):
    rc = getattr(_lib.lib(), name)(*args, None)
    text = _lib.lib().g4_last_error().decode()
    assert rc in codes and re.search(match, text) and name in text, (rc, text)


# --- packed prompts ----------------------------------------------------------------------------------------------


def _packed(**kw):
    base = dict(tokens=100, kv_heads=2, group=4, head_dim=256, window=0, k_stride=128, starts=AT, q=AT, k=AT, vt=AT, out=AT)
    return [ctypes.byref(_lib.G4PackedPrefillArgs(**{**base, **kw}))]


@pytest.mark.parametrize("override,match", [
    (dict(tokens=0), "tokens"), (dict(kv_heads=0), "kv_heads"), (dict(group=0), "group"), (dict(group=65), "group"),
    (dict(window=-1), "window"), (dict(head_dim=96), "head_dim"), (dict(head_dim=32), "head_dim"),
    (dict(k_stride=64), "k_stride"), (dict(k_stride=130), "k_stride"), (dict(starts=None), "NULL"), (dict(out=None), "NULL"),
    (dict(q=AT + 8), "aligned"), (dict(vt=AT + 2), "aligned"),
    (dict(tokens=1 << 23, k_stride=1 << 23), "too many"),  # a head's keys of 2^32 bytes
    (dict(tokens=1 << 25, k_stride=1 << 25, head_dim=64, group=64), "too many"),  # 2^31 rows
    (dict(tokens=1 << 21, k_stride=1 << 21, kv_heads=1 << 13), "too many"),  # a grid of 2^32 threads
    (dict(longest=-1), "longest"),
])
def test_packed_attention_refuses(override, match):
    _refused("g4_packed_prefill_attention", _packed(**override), match)


def test_packed_attention_refuses_a_short_workspace():
    few = dict(tokens=1000, k_stride=1024, head_dim=64, kv_heads=1)
    need = _lib.lib().g4_packed_prefill_workspace_size(*_packed(**few))
    assert need > 0 and _lib.lib().g4_packed_prefill_workspace_size(None) == 0
    for none in (dict(longest=100), dict(window=512), dict(tokens=700), dict(kv_heads=64, window=500), dict(kv_heads=64, longest=224)):
        assert _lib.lib().g4_packed_prefill_workspace_size(*_packed(**{**few, **none})) == 0
    # 2048 workgroups of 128 rows, 32 to a head: the order of 8 runs of them
    assert _lib.lib().g4_packed_prefill_workspace_size(*_packed(**{**few, "kv_heads": 64})) == 32
    for override in (dict(), dict(workspace=AT), dict(workspace=AT, workspace_bytes=need - 1), dict(workspace_bytes=need)):
        _refused("g4_packed_prefill_attention", _packed(**few, **override), "workspace", (_lib.G4_ERR_WORKSPACE,))
    _refused("g4_packed_prefill_attention", _packed(**few, workspace=AT + 4, workspace_bytes=need), "aligned")


@pytest.mark.parametrize("args,match", [((0, AT, 5, AT), "0 sequences"), ((2, None, 5, AT), "NULL"), ((2, AT, 0, AT), "0 tokens"),
                                        ((2, AT, 5, None), "NULL"), ((2, AT, 2 ** 31 - 1, AT), "tokens")])
def test_packed_starts_refuses(args, match):
    _refused("g4_packed_starts", args, match)


# --- the pool ------------------------------------------------------------------------------------------------------


def _layers(n=2, **kw):
    base = dict(format=_lib.G4_PAGES_E4M3, num_pages=8, kv_heads=2, head_dim=256, page_size=64, key=AT, value=AT, key_scale=AT,
                value_scale=AT)
    return (_lib.G4PagedCache * n)(*[_lib.G4PagedCache(**{**base, **(kw if i == n - 1 else {})}) for i in range(n)])


def _pool_table(**kw):
    return _lib.G4PageTable(**{**dict(rows=3, max_pages=4, stride=4, entries=AT), **kw})


def _reserve(table=None, **kw):
    base = dict(num_pages=8, page_size=64, table=_pool_table(**(table or {})), lengths=AT, refs=AT, shortage=AT, workspace=AT,
                workspace_bytes=1 << 30)
    return _lib.G4PagedReserveArgs(**{**base, **kw})


def _free(table=None, **kw):
    return _lib.G4PagedFreeArgs(**{**dict(num_pages=8, page_size=64, table=_pool_table(**(table or {})), keep=AT, refs=AT), **kw})


def _fork(table=None, out=None, layers=None, **kw):
    base = dict(layers=ctypes.addressof(layers), n_layers=len(layers), table=_pool_table(**(table or {})),
                out=_pool_table(**{**dict(entries=1 << 20), **(out or {})}), parents=AT, lengths=AT, refs=AT, shortage=AT, workspace=AT,
                workspace_bytes=1 << 30)
    return _lib.G4PagedForkArgs(**{**base, **kw})


def _compact(table=None, layers=None, **kw):
    base = dict(layers=ctypes.addressof(layers), n_layers=len(layers), table=_pool_table(**(table or {})), refs=AT, live=AT, workspace=AT,
                workspace_bytes=1 << 30)
    return _lib.G4PagedCompactArgs(**{**base, **kw})


BAD_TABLES = [(dict(rows=0), "page table"), (dict(max_pages=0), "page table"), (dict(stride=3), "page table"),
              (dict(entries=None), "page table"), (dict(rows=1 << 20, max_pages=1 << 12, stride=1 << 12), "entries")]


@pytest.mark.parametrize("table,match", BAD_TABLES)
def test_the_pool_refuses_bad_tables(table, match):
    layers = _layers()
    _refused("g4_paged_reserve", [ctypes.byref(_reserve(table))], match)
    _refused("g4_paged_free", [ctypes.byref(_free(table))], match)
    _refused("g4_paged_fork", [ctypes.byref(_fork(table, layers=layers))], match)
    _refused("g4_paged_fork", [ctypes.byref(_fork(out=table, layers=layers))], match)
    _refused("g4_paged_compact", [ctypes.byref(_compact(table, layers=layers))], match)


@pytest.mark.parametrize("make,name,override,match", [
    (_reserve, "g4_paged_reserve", dict(num_pages=0), "num_pages"),
    (_reserve, "g4_paged_reserve", dict(num_pages=2 ** 31 - 1), "num_pages"),
    (_reserve, "g4_paged_reserve", dict(page_size=48), "page_size"),
    (_reserve, "g4_paged_reserve", dict(refs=None), "refs"),
    (_reserve, "g4_paged_reserve", dict(lengths=None), "lengths"),
    (_reserve, "g4_paged_reserve", dict(shortage=None), "shortage"),
    (_free, "g4_paged_free", dict(page_size=2048), "page_size"),
    (_free, "g4_paged_free", dict(keep=None), "keep"),
    (_free, "g4_paged_free", dict(refs=None), "refs"),
])
def test_the_pool_refuses_bad_calls(make, name, override, match):
    _refused(name, [ctypes.byref(make(**override))], match)


@pytest.mark.parametrize("override,match", [
    (dict(format=3), "format"), (dict(num_pages=9), "layer 1"), (dict(page_size=32), "layer 1"), (dict(key=None), "NULL"),
    (dict(head_dim=96), "head_dim"), (dict(kv_heads=1 << 20), "heads"), (dict(key_scale=None), "key_scale"),
])
def test_the_pool_refuses_bad_layers(override, match):
    layers = _layers(**override)
    _refused("g4_paged_fork", [ctypes.byref(_fork(layers=layers))], match)
    _refused("g4_paged_compact", [ctypes.byref(_compact(layers=layers))], match)
    _refused("g4_paged_copy", [ctypes.addressof(layers), len(layers), 3, AT, AT], match)


def test_the_pool_refuses_nothing_to_do_and_overlaps():
    layers = _layers()
    for args in ((None, 2, 3, AT, AT), (ctypes.addressof(layers), 0, 3, AT, AT), (ctypes.addressof(layers), 2, 0, AT, AT),
                 (ctypes.addressof(layers), 2, 3, None, AT)):
        _refused("g4_paged_copy", args, "layers|pairs")
    for key, match in (("parents", "parents"), ("lengths", "lengths"), ("shortage", "shortage"), ("refs", "refs")):
        _refused("g4_paged_fork", [ctypes.byref(_fork(layers=layers, **{key: None}))], match)
    _refused("g4_paged_fork", [ctypes.byref(_fork(layers=layers, out=dict(entries=AT + 44)))], "overlaps")  # 12 entries of 4 bytes
    _refused("g4_paged_fork", [ctypes.byref(_fork(layers=layers, table=dict(max_pages=1 << 26, stride=1 << 26),
                                                  out=dict(max_pages=1 << 26, stride=1 << 26, entries=1 << 40)))], "2\\^31")
    _refused("g4_paged_compact", [ctypes.byref(_compact(layers=layers, live=None))], "live")
    for name in ("g4_paged_reserve", "g4_paged_fork", "g4_paged_free", "g4_paged_compact", "g4_packed_prefill_attention",
                 "g4_verify_draft"):
        assert getattr(_lib.lib(), name)(None, None) == _lib.G4_ERR_INVALID


def test_workspaces_are_checked():
    L, layers = _lib.lib(), _layers()
    for make, name in ((lambda **kw: _reserve(**kw), "g4_paged_reserve"), (lambda **kw: _fork(layers=layers, **kw), "g4_paged_fork"),
                       (lambda **kw: _compact(layers=layers, **kw), "g4_paged_compact"), (lambda **kw: _verify(**kw), "g4_verify_draft")):
        need = getattr(L, name + "_workspace_size")(ctypes.byref(make()))
        assert need > 0 and getattr(L, name + "_workspace_size")(None) == 0
        _refused(name, [ctypes.byref(make(workspace=None))], "workspace", (_lib.G4_ERR_WORKSPACE,))
        _refused(name, [ctypes.byref(make(workspace_bytes=need - 1))], "workspace", (_lib.G4_ERR_WORKSPACE,))
        _refused(name, [ctypes.byref(make(workspace=AT + 8))], "aligned")


# --- verification ----------------------------------------------------------------------------------------------------


def _verify(**kw):
    base = dict(dtype=_lib.G4_DTYPE_BF16, batch=2, drafts=3, vocab=100, logits=AT, batch_stride=400, row_stride=100, draft_logits=None,
                draft_batch_stride=300, draft_row_stride=100, draft_tokens=AT, draft_lengths=None, uniforms=AT, noise=AT,
                noise_stride=100, temperature=1.0, token_out=AT, count_out=AT, logp_out=AT, workspace=AT, workspace_bytes=1 << 30)
    return _lib.G4VerifyArgs(**{**base, **kw})


@pytest.mark.parametrize("override,match", [
    (dict(dtype=5), "dtype"), (dict(batch=0), "batch"), (dict(drafts=0), "drafts"), (dict(drafts=64), "drafts"),
    (dict(vocab=0), "vocab"), (dict(vocab=2 ** 31 - 1), "vocab"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-9), "temperature"), (dict(logits=None), "NULL"),
    (dict(draft_tokens=None), "NULL"), (dict(count_out=None), "NULL"), (dict(uniforms=None), "uniforms"), (dict(noise=None), "noise"),
    (dict(logits=AT + 1), "aligned"), (dict(row_stride=99), "strides"), (dict(batch_stride=99), "strides"),
    (dict(noise_stride=99), "strides"), (dict(draft_logits=AT, draft_row_stride=99), "strides"),
    (dict(draft_logits=AT, draft_batch_stride=99), "strides"), (dict(noise=AT + 2), "aligned"),
    (dict(batch=1 << 20, drafts=63, batch_stride=6400, workspace_bytes=1 << 50), "too many"),
])
def test_verify_refuses(override, match):
    _refused("g4_verify_draft", [ctypes.byref(_verify(**override))], match)


# --- the Python front end ------------------------------------------------------------------------------------------


def _i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def _bf(*s):
    return torch.zeros(s, dtype=torch.bfloat16)


def _error(match, call, *a, kind=ValueError, **kw):
    with pytest.raises(kind, match=match):
        call(*a, **kw)


def test_front_end_of_packed_attention():
    q, k, vt, starts = _bf(70, 2, 4, 64), _bf(*key_shape(1, 2, 128, 64)), _bf(1, 2, 16, 64, 8), _i32(70)
    call = kernels.packed_prefill_attention
    _error("device tensors", call, q, k, vt, starts)
    _error("q must", call, q.float(), k, vt, starts)
    _error("q must", call, q[:, :, ::2], k, vt, starts)
    _error("q must", call, q[0], k, vt, starts)
    _error("layouts", call, q, k[0], vt, starts)
    _error("do not match", call, q, _bf(*key_shape(2, 2, 128, 64)), vt, starts)
    _error("do not match", call, q, _bf(*key_shape(1, 2, 64, 64)), _bf(1, 2, 8, 64, 8), starts)
    _error("do not match", call, q, k, _bf(1, 2, 16, 32, 8), starts)
    _error("bfloat16", call, q, k.float(), vt, starts)
    _error("starts must", call, q, k, vt, starts.long())
    _error("starts must", call, q, k, vt, starts[:60])
    _error("window", call, q, k, vt, starts, window=-2)
    _error("longest", call, q, k, vt, starts, longest=-1)
    _error("out must", call, q, k, vt, starts, out=_bf(70, 2, 4, 32))
    _error("cu_seqlens", kernels.packed_starts, starts.long(), 5)
    _error("cu_seqlens", kernels.packed_starts, starts[:1], 5)
    _error("tokens", kernels.packed_starts, starts, 0)
    _error("device tensors", kernels.packed_starts, starts, 5)


def test_front_end_of_the_pool():
    layer, other = new_paged_layer(4, 2, 64, 32, device="cpu"), new_paged_layer(5, 2, 64, 32, device="cpu")
    refs, table, n = _i32(4), _i32(3, 2), _i32(3)
    calls = [(lambda refs=refs, table=table, n=n, layers=None: kernels.paged_reserve(refs, table, n, page_size=32)),
             (lambda refs=refs, table=table, n=n, layers=None: kernels.paged_free(refs, table, n, page_size=32)),
             (lambda refs=refs, table=table, n=n, layers=(layer,): kernels.paged_fork(layers, refs, table, _i32(6), n)),
             (lambda refs=refs, table=table, n=n, layers=(layer,): kernels.paged_compact(layers, refs, table))]
    for i, call in enumerate(calls):
        _error("device tensors", call)
        _error("refs", call, refs=refs.long())
        _error("refs", call, refs=_i32(0))
        _error("page_table", call, table=table.long())
        _error("page_table", call, table=table[:, :0])
        _error("page_table", call, table=_i32(2, 3).t())
        if i < 3:
            _error("int32 \\[3\\]", call, n=n[:2])
            _error("int32 \\[3\\]", call, n=n.long())
        if i > 1:
            _error("refs has", call, refs=_i32(7))
            _error("empty", call, layers=())
            _error("share no tables", call, layers=(layer, other))
    _error("parents", kernels.paged_fork, (layer,), refs, table, _i32(0), n)
    _error("parents", kernels.paged_fork, (layer,), refs, table, _i32(6).long(), n)
    _error("src", kernels.paged_copy, (layer,), _i32(0), _i32(0))
    _error("targets", kernels.paged_copy, (layer,), _i32(3), _i32(4))
    _error("dst", kernels.paged_copy, (layer,), _i32(3), _i32(3).long())
    _error("device tensors", kernels.paged_copy, (layer,), _i32(3), _i32(3))


def test_front_end_of_the_verification():
    x, d, u, w = _bf(2, 4, 50), _i32(2, 3), torch.zeros(2, 3), torch.zeros(2, 50)
    call = lambda x=x, d=d, u=u, w=w, **kw: kernels.verify_draft(x, d, u, w, **{**dict(temperature=1.0), **kw})  # noqa: E731
    _error("device tensors", call)
    _error("logits must", call, x=x[0])
    _error("logits must", call, x=x[:, :1])
    _error("unsupported dtype", call, x=x.half(), kind=TypeError)
    _error("logits: strides", call, x=_bf(2, 50, 4).transpose(1, 2))
    _error("logits: strides", call, x=x[:, :1].expand(2, 4, 50))
    _error("draft_tokens", call, d=d.long())
    _error("draft_tokens", call, d=d[:, :2])
    _error("uniforms", call, u=u.double())
    _error("uniforms", call, u=torch.zeros(2, 4))
    _error("noise", call, w=torch.zeros(2, 49))
    _error("noise", call, w=torch.zeros(50, 2).t())
    _error("draft_logits: shape", call, draft_logits=x)
    _error("draft_logits are", call, draft_logits=x[:, :3].float(), kind=TypeError)
    _error("draft_lengths", call, draft_lengths=_i32(3))


@pytest.mark.parametrize("capacity,window,ps", [(1, 1, 32), (200, 40, 32), (5000, 512, 64), (64, 512, 64), (4096, 33, 32)])
def test_page_counts(capacity, window, ps):
    """A ring has the pages that a window touches at most, wherever it starts."""

    width, cycle = page_counts(capacity, window, ps)
    assert width == -(-capacity // ps)
    touched = max((p + window - 1) // ps - p // ps + 1 for p in range(ps))
    assert cycle == min(width, touched)
