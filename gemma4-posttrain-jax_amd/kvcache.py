"""Device KV cache in the layout the gfx950 kernels read (mirrors model.py:238-255, 557-568).

Per non-shared layer: ``key [B, Hkv, slot_stride / 32, D / KR, 2, 16, KR]`` (KR = min(D, 32)) and ``value_t
[B, Hkv, slot_stride / 8, D, 8]`` in the parameter dtype: the values in groups of 8 slots, each
group stored d-major, so the 8 slots of one value dim are contiguous (one 16-byte MFMA operand in
bf16) and one slot's D values lie in one 8 * D-element span (an append touches D / 8 cache lines).
``value_dmajor()`` gives the plain transposed ``[B, Hkv, D, slot_stride]`` view. The keys of each
32-slot chunk are stored in the order of the attention MFMA's A operand (block (chunk, dims/32, bb)
holds 16 lanes x 32 dims, lane col = slot 8 (col >> 2) + 4 bb + (col & 3) of the chunk), so one
operand load reads one contiguous KiB; ``key_slots()`` gives slot-major ``[B, Hkv, slot_stride, D]``.
Sliding layers
keep a ring of ``Wc = min(window, C)`` slots, global layers ``C = prompt + new`` slots, kv-shared
layers ``None`` (model.py:557-568). ``slot_stride`` rounds the slot count up to 64 so every row
is 128-byte aligned. ``key_mask [B, C]`` (bool, 1 byte per entry) records which absolute
positions hold real tokens; ``length`` is the number of positions written so far (the
reference's scalar ``KVCache.length``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .config import FULL, SLIDING, Gemma4TextConfig, is_kv_shared, layer_head_dim, layer_kv_heads


def slot_stride_for(capacity: int) -> int:
    return (capacity + 63) // 64 * 64


def key_shape(batch: int, heads: int, slots: int, head_dim: int) -> tuple:
    """Shape of the operand-ordered key layout: ``[B, H, slots / 32, D / KR, 2, 16, KR]``,
    KR = min(D, 32) dims per run (slots a multiple of 32)."""

    kr = min(head_dim, 32)
    return (batch, heads, slots // 32, head_dim // kr, 2, 16, kr)


def group_keys(k: torch.Tensor) -> torch.Tensor:
    """Slot-major keys ``[B, H, Sp, D]`` (Sp a multiple of 32) -> the kernels' operand-ordered
    layout (``key_shape``; contiguous copy). Slot 8 a + 4 bb + c of a chunk goes to half bb, lane
    4 a + c."""

    B, H, Sp, D = k.shape
    kr = min(D, 32)
    t = k.reshape(B, H, Sp // 32, 4, 2, 4, D // kr, kr).permute(0, 1, 2, 6, 4, 3, 5, 7)
    return t.reshape(key_shape(B, H, Sp, D)).contiguous()


def ungroup_keys(kt: torch.Tensor) -> torch.Tensor:
    """The operand-ordered key layout -> slot-major ``[B, H, Sp, D]`` (copy)."""

    B, H, C, NR = kt.shape[:4]
    kr = kt.shape[6]
    return kt.reshape(B, H, C, NR, 2, 4, 4, kr).permute(0, 1, 2, 5, 4, 6, 3, 7).reshape(B, H, C * 32, NR * kr)


def group_values(v: torch.Tensor) -> torch.Tensor:
    """Slot-major values ``[B, H, Sp, D]`` (Sp a multiple of 8) -> the kernels' grouped layout
    ``[B, H, Sp / 8, D, 8]`` (contiguous copy)."""

    B, H, Sp, D = v.shape
    return v.reshape(B, H, Sp // 8, 8, D).transpose(3, 4).contiguous()


def ungroup_values(vt: torch.Tensor) -> torch.Tensor:
    """The grouped layout ``[B, H, G, D, 8]`` -> slot-major ``[B, H, 8 G, D]`` (copy)."""

    B, H, G, D, _ = vt.shape
    return vt.transpose(3, 4).reshape(B, H, G * 8, D)


class LayerKVCache(NamedTuple):
    key: torch.Tensor  # [B, Hkv, slot_stride / 32, D / KR, 2, 16, KR], KR = min(D, 32)
    value_t: torch.Tensor  # [B, Hkv, slot_stride / 8, D, 8]
    capacity: int  # logical slots: C (linear) or Wc (ring)
    ring: bool

    @property
    def slot_stride(self) -> int:
        return self.key.shape[2] * 32

    @property
    def head_dim(self) -> int:
        return self.key.shape[3] * self.key.shape[6]

    def key_slots(self) -> torch.Tensor:
        """The keys as slot-major ``[B, Hkv, slot_stride, D]`` (a copy)."""

        return ungroup_keys(self.key)

    def set_keys(self, k: torch.Tensor) -> None:
        """Write ``k [B, Hkv, capacity, D]`` (slot major) into slots ``[0, capacity)`` in place."""

        full = self.key_slots()
        full[:, :, : k.shape[2]] = k
        self.key.copy_(group_keys(full))

    def value_dmajor(self) -> torch.Tensor:
        """The values as ``[B, Hkv, D, slot_stride]`` (value dim major; a copy)."""

        B, H, G, D, _ = self.value_t.shape
        return self.value_t.permute(0, 1, 3, 2, 4).reshape(B, H, D, G * 8)

    def set_values(self, v: torch.Tensor) -> None:
        """Write ``v [B, Hkv, capacity, D]`` (slot major) into slots ``[0, capacity)`` in place."""

        B, H, C, D = v.shape
        full = self.value_t.permute(0, 1, 2, 4, 3).reshape(B, H, -1, D)  # [B, H, slot_stride, D] copy
        full[:, :, :C] = v
        self.value_t.copy_(full.reshape(B, H, -1, 8, D).permute(0, 1, 2, 4, 3))

    def reference_layout(self) -> tuple[torch.Tensor, torch.Tensor]:
        """``(key, value)`` as the reference's ``[B, capacity, Hkv, D]`` arrays (copies)."""

        k = self.key_slots()[:, :, : self.capacity].permute(0, 2, 1, 3).contiguous()
        v = self.value_dmajor()[:, :, :, : self.capacity].permute(0, 3, 1, 2).contiguous()
        return k, v


PAGE_SIZES = (32, 64, 128, 256, 512, 1024)


def paged_key_shape(pages: int, heads: int, page_size: int, head_dim: int, e4m3: bool) -> tuple:
    """Shape of a layer's key pages: ``[P, H, page / 32, D / KR, 2, 16, KR]``, the dense key layout per 32-slot
    chunk with runs of KR = 32 (bf16) or 64 (e4m3) dims."""

    kr = 64 if e4m3 else 32
    return (pages, heads, page_size // 32, head_dim // kr, 2, 16, kr)


class PagedLayerCache(NamedTuple):
    """One layer's K/V in pages of ``page_size`` positions (g4_paged_append, g4_paged_decode_attention,
    g4_paged_read), in bf16, or in e4m3 with one power-of-two scale per slot and head of each of K and V.
    Which pages a row has, and in which order, is the caller's ``page_table [B, M]`` (int32): position p of
    row b is slot ``p % page_size`` of page ``page_table[b, p // page_size]``, and an entry outside
    ``[0, P)`` stands for no page. Rows may share pages."""

    key: torch.Tensor  # paged_key_shape(...), bf16 or float8_e4m3fn
    value: torch.Tensor  # [P, Hkv, page / 8, D, 8]
    key_scale: torch.Tensor | None = None  # e4m3: [P, Hkv, page] float8_e8m0fnu
    value_scale: torch.Tensor | None = None

    @property
    def num_pages(self) -> int:
        return self.value.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.value.shape[1]

    @property
    def page_size(self) -> int:
        return self.value.shape[2] * 8

    @property
    def head_dim(self) -> int:
        return self.value.shape[3]

    @property
    def e4m3(self) -> bool:
        return self.value.dtype == torch.float8_e4m3fn


def new_paged_layer(num_pages: int, kv_heads: int, head_dim: int, page_size: int, *, e4m3: bool = False,
                    device="cuda") -> PagedLayerCache:
    """A zero-filled ``PagedLayerCache`` of ``num_pages`` pages, bf16 or e4m3."""

    if num_pages <= 0 or kv_heads <= 0:
        raise ValueError(f"num_pages and kv_heads must be positive, got {num_pages} and {kv_heads}")
    if head_dim not in (64, 128, 256, 512):
        raise ValueError(f"pages hold head dims 64, 128, 256 or 512, got {head_dim}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    key = paged_key_shape(num_pages, kv_heads, page_size, head_dim, e4m3)
    value = (num_pages, kv_heads, page_size // 8, head_dim, 8)
    if not e4m3:
        return PagedLayerCache(*(torch.zeros(s, dtype=torch.bfloat16, device=device) for s in (key, value)))
    key, value = (torch.zeros(s, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for s in (key, value))
    scales = (torch.full((num_pages, kv_heads, page_size), 127, dtype=torch.uint8, device=device)
              .view(torch.float8_e8m0fnu) for _ in range(2))
    return PagedLayerCache(key, value, *scales)


class KVCache(NamedTuple):
    layers: tuple  # LayerKVCache | None per layer
    key_mask: torch.Tensor  # [B, C] bool
    length: int


class PagedSpec(NamedTuple):
    """How ``init_paged_kv_cache`` lays out a cache: positions per page, and whether pages hold e4m3 (one byte
    per element and one scale per vector) instead of bf16."""

    page_size: int = 64
    e4m3: bool = False


class PagedKVCache(NamedTuple):
    """A model's cache in pages. Rows hold their real tokens only, in the order in which they came: left pads and
    the masked steps of a finished row take no slot, and a sliding layer's window is over what the row holds.
    Sliding layers share ``window_table``, whose rows cycle through the few pages that a window touches; global
    layers ``page_table``. ``length`` counts the physical positions processed, pads included, as
    ``KVCache.length``.

    ``held`` are the rows' token counts, so the place of their next tokens. A prefill sets it. ``None`` (an empty
    cache, or one whose pages the caller fills by ``kernels.paged_append``) leaves the places to the caller: a
    step's token goes to ``position_ids``, and every place below it has to be filled. ``pad`` are the pads that
    all rows of the prefill began with: the longest row holds at most ``length - pad`` tokens, and a step is
    refused where that is ``capacity``.

    ``refs`` counts the entries of ``page_table`` that hold each page, where rows share pages (``prefill_group``): what
    ``kernels.paged_free`` takes to let rows go that have ended, and ``kernels.paged_compact`` with the global layers. The
    rings are each row's own."""

    layers: tuple  # PagedLayerCache | None per layer
    page_table: torch.Tensor  # [B, M] int32, of the global layers
    window_table: torch.Tensor  # [B, M] int32, of the sliding layers
    length: int
    held: torch.Tensor | None = None  # [B] int32
    pad: int = 0
    refs: torch.Tensor | None = None  # [P] int32, of the global layers' pages

    @property
    def batch(self) -> int:
        return self.page_table.shape[0]

    @property
    def device(self) -> torch.device:
        return self.page_table.device

    @property
    def capacity(self) -> int:
        """Positions that a row can hold."""

        return self.page_table.shape[1] * next(x for x in self.layers if x is not None).page_size

    def check_room(self, length: int) -> None:
        """ValueError if a row may be full after ``length`` physical positions: another token would have no page."""

        if length - self.pad >= self.capacity:
            raise ValueError(f"no place for another token: the cache holds {self.capacity} positions, and "
                             f"{length - self.pad} were processed")


def page_counts(capacity: int, window: int, page_size: int) -> tuple[int, int]:
    """Pages of a row of ``capacity`` positions, and those that a sliding layer's ring takes of them: as many as ``window``
    positions touch at most."""

    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    width = (capacity + page_size - 1) // page_size
    return width, min(width, (window + page_size - 2) // page_size + 1)


def init_paged_kv_cache(config: Gemma4TextConfig, batch_size: int, capacity: int, spec: PagedSpec = PagedSpec(),
                        device="cuda") -> PagedKVCache:
    """``init_kv_cache`` in pages: every row gets the pages of ``capacity`` positions on global layers and those
    that a window can touch on sliding ones, ``None`` on kv-shared layers; zero-filled."""

    if batch_size <= 0 or capacity <= 0:
        raise ValueError(f"batch_size and capacity must be positive, got {batch_size} and {capacity}")
    ps = spec.page_size
    width, cycle = page_counts(capacity, config.sliding_window, ps)
    layers = []
    for i in range(config.num_hidden_layers):
        if is_kv_shared(config, i):
            layers.append(None)
            continue
        pages = batch_size * (cycle if config.layer_types[i] == SLIDING else width)
        layers.append(new_paged_layer(pages, layer_kv_heads(config, i), layer_head_dim(config, i), ps, e4m3=spec.e4m3,
                                      device=device))
    rows = torch.arange(batch_size, dtype=torch.int32, device=device)[:, None]
    entry = torch.arange(width, dtype=torch.int32, device=device)[None, :]
    return PagedKVCache(tuple(layers), rows * width + entry, rows * cycle + entry % cycle, 0)


def new_layer_cache(batch: int, kv_heads: int, head_dim: int, capacity: int, ring: bool, dtype, device) -> LayerKVCache:
    ss = slot_stride_for(capacity)
    key = torch.zeros(key_shape(batch, kv_heads, ss, head_dim), dtype=dtype, device=device)
    value_t = torch.zeros((batch, kv_heads, ss // 8, head_dim, 8), dtype=dtype, device=device)
    return LayerKVCache(key, value_t, capacity, ring)


def init_kv_cache(config: Gemma4TextConfig, batch_size: int, capacity: int, dtype, device="cuda") -> KVCache:
    """model.py:557-568: bounded rings on sliding layers, full capacity on global layers,
    ``None`` on kv-shared layers; zero-filled."""

    layers = []
    for i in range(config.num_hidden_layers):
        if is_kv_shared(config, i):
            layers.append(None)
            continue
        ring = config.layer_types[i] == SLIDING
        cap = min(config.sliding_window, capacity) if ring else capacity
        layers.append(new_layer_cache(batch_size, layer_kv_heads(config, i), layer_head_dim(config, i), cap, ring,
                                      dtype, device))
    key_mask = torch.zeros((batch_size, capacity), dtype=torch.bool, device=device)
    return KVCache(tuple(layers), key_mask, 0)


__all__ = ["LayerKVCache", "KVCache", "PagedLayerCache", "PagedKVCache", "PagedSpec", "PAGE_SIZES", "new_paged_layer",
           "page_counts", "paged_key_shape", "init_kv_cache", "init_paged_kv_cache", "new_layer_cache", "slot_stride_for", "key_shape",
           "group_keys", "ungroup_keys", "group_values", "ungroup_values", "FULL", "SLIDING"]
