"""The paged cache: device memory for the pages, host bookkeeping for who holds which.

Bookkeeping (free lists, block tables, slots) is the C++ ``CacheManager``
(``csrc/host/cache_manager.hpp``). This class adds the device side: for every
group of layer calls with the same needs, a pool ``K`` and ``V`` of shape
``[calls, num_pages, kv_heads, page_size, head_dim]``, and for every call with
state of fixed size an array ``[max_requests, *shape]`` indexed by the request's
slot. The reference keeps both per sequence (garuda/src/cache/mod.rs:221-241,
:610-619, :630-648); here they are pools shared by all requests.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from ..csrc.build import load_host_module
from ..parts.base import LayerCache, PagedKV, PagedLatent, FixedState


@dataclass
class CacheConfig:
    page_size: int = 32                 # positions per page (garuda/src/llama/mod.rs:483 uses 32)
    num_pages: Optional[int] = None     # pages per group; None: from max_tokens
    max_tokens: Optional[int] = None    # positions the pool holds per group
    max_requests: int = 4               # request slots (garuda/src/config/mod.rs:166-167)
    max_positions: int = 2048           # positions one request may hold


class PagedCache:
    def __init__(self, model, config: CacheConfig, dtype: torch.dtype, device, allocate: bool = True, float8: bool = False):
        """``float8``: the pages hold 8-bit numbers (E4M3) with a 32-bit scale per page and key/value head, ``k_scales`` and
        ``v_scales`` ``[calls, num_pages, kv_heads]`` of every group; states of fixed size stay as they are."""
        host = load_host_module()
        self.host_module = host
        self.config = config
        self.model = model
        self.dtype, self.device = dtype, torch.device(device)
        self.float8 = bool(float8)
        if float8 and any(isinstance(g.need, PagedLatent) for g in model.cache_groups):
            raise ValueError("pages in 8 bits hold keys and values, not latent rows")
        page_dtype = torch.float8_e4m3fn if float8 else dtype
        ps = config.page_size
        if config.num_pages is not None:
            pages = int(config.num_pages)
        elif config.max_tokens is not None:
            pages = (int(config.max_tokens) + ps - 1) // ps
        else:
            raise ValueError("the cache needs num_pages or max_tokens")
        self.groups = model.cache_groups
        self.manager = host.CacheManager(
            [host.GroupConfig(pages, g.need.window or 0, getattr(g.need, "keep_first", 0) or 0,
                              getattr(g.need, "chunk", 0) or 0) for g in self.groups],
            ps, config.max_requests, config.max_positions)
        self.page_size = ps
        self.table_width = self.manager.max_pages_per_request
        # device memory
        self.k_pools: List[torch.Tensor] = []
        self.v_pools: List[torch.Tensor] = []
        self.k_scales: List[torch.Tensor] = []
        self.v_scales: List[torch.Tensor] = []
        self.call_group: Dict[object, tuple] = {}
        for gi, g in enumerate(self.groups):
            if isinstance(g.need, PagedLatent):
                # one vector per position, shared by the heads: a single pool (there is no value pool)
                shape = (len(g.calls), pages, 1, ps, g.need.width)
                if allocate:
                    self.k_pools.append(torch.zeros(shape, dtype=dtype, device=self.device))
                    self.v_pools.append(None)
            else:
                shape = (len(g.calls), pages, g.need.kv_heads, ps, g.need.head_dim)
                v_shape = shape[:-1] + (g.need.value_dim or g.need.head_dim,)
                if allocate:
                    self.k_pools.append(torch.zeros(shape, dtype=page_dtype, device=self.device))
                    self.v_pools.append(torch.zeros(v_shape, dtype=page_dtype, device=self.device))
                    if float8:
                        self.k_scales.append(torch.zeros(shape[:3], dtype=torch.float32, device=self.device))
                        self.v_scales.append(torch.zeros(shape[:3], dtype=torch.float32, device=self.device))
            for j, call in enumerate(g.calls):
                self.call_group[call] = (gi, j)
        self.states: Dict[object, torch.Tensor] = {}
        for call in model.state_calls:
            need: FixedState = model.need_at(call)
            if allocate:
                self.states[call] = torch.zeros((config.max_requests, *need.shape), dtype=need.dtype,
                                                device=self.device)

    # ---- request lifecycle -------------------------------------------------
    def acquire(self, request: int) -> int:
        """A slot for a new request. Its fixed-size state is zeroed by the step that runs the
        request's first token (``reset_states``), so that it makes no difference who took the
        slot: this call, or a scheduler working on the bookkeeping directly."""
        return self.manager.acquire(request)

    def reset_states(self, slots: Sequence[int]) -> None:
        """Fixed-size state of these slots back to zero, in every layer call that keeps some
        (garuda/src/cache/mod.rs:719-743: a sequence's state starts as zeros)."""
        if not self.states or not slots:
            return
        for s in self.states.values():
            for slot in slots:
                s[slot].zero_()

    def release(self, request: int) -> None:
        self.manager.release(request)

    def bytes_per_position(self) -> int:
        if self.float8:         # and a page's two scales a head
            return sum(len(g.calls) * (g.need.kv_heads * (g.need.head_dim + (g.need.value_dim or g.need.head_dim))
                                       + -(-8 * g.need.kv_heads // self.page_size)) for g in self.groups)
        item = self.dtype.itemsize
        return sum(len(g.calls) * (g.need.width if isinstance(g.need, PagedLatent)
                                   else g.need.kv_heads * (g.need.head_dim + (g.need.value_dim or g.need.head_dim)))
                   * item for g in self.groups)

    # ---- views for a step ------------------------------------------------------
    def layer_caches(self, block_tables: Sequence[torch.Tensor]) -> List[Optional[LayerCache]]:
        """One ``LayerCache`` per entry of the model's run order, over the given
        device block tables (one per group, rows in the batch's request order)."""
        out: List[Optional[LayerCache]] = []
        order = self.model.spec.order

        def one(need, key, writes):
            if need is None:
                return None
            if isinstance(need, (PagedKV, PagedLatent)):
                gi, j = self.call_group[key]
                v_pool = self.v_pools[gi]
                return LayerCache(need=need, k=self.k_pools[gi][j], v=None if v_pool is None else v_pool[j],
                                  block_table=block_tables[gi], page_size=self.page_size, writes=writes,
                                  k_scale=self.k_scales[gi][j] if self.float8 else None,
                                  v_scale=self.v_scales[gi][j] if self.float8 else None)
            return LayerCache(need=need, state=self.states[key], writes=writes)

        for i, call in enumerate(order):
            need = self.model.call_need[i]
            src = i if call.reads_cache_of is None else call.reads_cache_of
            writes = call.reads_cache_of is None
            if isinstance(need, tuple):
                # a mixer made of several mixers: a cache per member
                out.append(LayerCache(need=need, writes=writes,
                                      parts=tuple(one(n, (src, k), writes) for k, n in enumerate(need))))
            else:
                out.append(one(need, src, writes))
        return out
