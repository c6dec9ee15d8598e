"""Decoding along several branches: the checking wrappers of its kernels.

A step may bring a *tree* of drafted tokens per request instead of a stretch: token 0 is the request's last one, which the cache does not hold
yet, and ``parents`` names for every other the token of the same request that it continues. A step with trees goes: ``tree_layout`` once; in every
layer the projections' queries and keys are turned by its positions (``CudaOps.rope_inplace``), keys and values go behind the request's context in the
order of the tokens' numbers (``rope_kv_append`` with those places and no rotation of its own), and ``tree_attention`` reads them; behind the logits
``tree_accept`` keeps the tokens that the model would have chosen itself and moves what they left in the cache together.

*Beams* are requests of their own over shared pages: ``beam_select`` chooses how they go on, ``copy_entries`` gives a beam that goes on in several
ways a copy of its last page and of its states (``PagedCache.fork`` says which).
"""
from __future__ import annotations

import ctypes
import math
import struct
from array import array
from ctypes import c_char_p, c_int, c_longlong, c_void_p

import torch

from ..csrc.build import load_kernel_lib
from .checks import _TAG, KernelError, _need

_capturing = torch._C._cuda_isCurrentStreamCapturing

_SIGNATURES = {
    "gb_tree_layout": [c_void_p] * 5 + [c_int] * 4 + [c_void_p],
    "gb_tree_accept": [c_char_p],
    "gb_tree_attention_tc": [c_char_p],
    "gb_tree_attention_simple": [c_char_p],
    "gb_beam_select": [c_char_p],
    "gb_copy_entries": [c_char_p],
    "gb_tree_attention_error_check": [],
    "gb_tree_attention_set_error_sink": [c_void_p],
    "gb_beam_select_error_check": [],
    "gb_beam_select_set_error_sink": [c_void_p],
    "gb_branches_error_check": [],
    "gb_branches_set_error_sink": [c_void_p],
}
# What the entry points of one argument take: the fields of their structures in order, eight bytes each (a call of two dozen arguments takes three
# microseconds, packing them half of one)
_TREE_CALL, _ACCEPT_CALL, _BEAM_CALL, _COPY_CALL = (struct.Struct(f) for f in ("=12Q13qd", "=11Q7q", "=8Q5q", "=4Q2q"))


class BranchOps:
    """What ``CudaOps`` has of branches. Everything is launched on torch's current stream; results do not depend on the order in which blocks
    finish. Scratch memory is the call's ``ws``, else that of the step that is running (``scratch_from``), else one that the set
    keeps for the stream; a call captured into a graph without ``ws`` has memory of its graph's own (and clears its counters in every replay). One
    ``ws`` is for one stream at a time, and not to be used on after a call that gave up a wait."""

    #: ``tree_layout`` and ``tree_accept`` take trees of up to this many tokens
    MOST_DRAFTED = 8192
    #: ``tree_attention`` reads requests of up to this many positions
    MOST_POSITIONS = 1 << 30
    #: ``copy_entries`` makes up to this many copies
    MOST_COPIES = 1024
    #: ``beam_select`` takes up to this many beams and chooses up to this many candidates
    MOST_BEAMS = 64

    @property
    def branch_lib(self):
        """The library of these kernels, compiled and loaded when a caller first needs it."""
        if self._branches is None:
            L = load_kernel_lib("garuda_branches")
            L.gb_last_error.restype = ctypes.c_char_p
            for name, argtypes in _SIGNATURES.items():
                fn = getattr(L, name)
                fn.argtypes, fn.restype = argtypes, c_int
            sizes = {"gb_tree_attention_scratch_bytes": [c_int, ctypes.POINTER(c_longlong)],
                     "gb_beam_select_scratch_bytes": [c_int] * 4 + [ctypes.POINTER(c_longlong)]}
            for name, argtypes in sizes.items():
                fn = getattr(L, name)
                fn.argtypes, fn.restype = argtypes, c_longlong
            self._branch_sizes, self._branch_scratch = {}, {}
            if any([sink(self.error_word.data_ptr()) for sink in (L.gb_tree_attention_set_error_sink, L.gb_beam_select_set_error_sink,
                                                                     L.gb_branches_set_error_sink)]):
                _need(False, "the library of branches could not be given the host's error word")
            self._branches = L
        return self._branches

    def _branch_memory(self, name, sizes, key, ws, stream):
        """Addresses of a call's scratch and counters (zero when they are made), and what keeps them; ``sizes`` is the library's function that
        gives their bytes."""
        known = self._branch_sizes.get((name, key))
        if known is None:
            if len(self._branch_sizes) > 4096:
                self._branch_sizes.clear()
            counter_bytes = c_longlong(0)
            nbytes = sizes(*key, ctypes.byref(counter_bytes))
            known = self._branch_sizes[name, key] = (nbytes, int(counter_bytes.value))
        nbytes, counter_bytes = known
        if ws is None:
            ws = self.step_ws
        if ws is not None:
            held = ws.get(name, (nbytes,), torch.uint8), ws.get(name + "_counters", (counter_bytes,), torch.uint8, zero=True)
        elif _capturing():
            held = torch.empty(nbytes, dtype=torch.uint8, device=self.device), torch.zeros(counter_bytes, dtype=torch.uint8, device=self.device)
        else:
            kept = self._branch_scratch.get((name, stream))
            if kept is None or kept[0] < nbytes or kept[1] < counter_bytes:
                if kept is not None:
                    nbytes, counter_bytes = max(nbytes, kept[0]), max(counter_bytes, kept[1])
                held = torch.empty(nbytes, dtype=torch.uint8, device=self.device), torch.zeros(counter_bytes, dtype=torch.uint8, device=self.device)
                kept = self._branch_scratch[name, stream] = (nbytes, counter_bytes, held[0].data_ptr(), held[1].data_ptr(), held)
            return kept[2:]
        return held[0].data_ptr(), held[1].data_ptr(), held

    def branch_error_code(self) -> int:
        """The code of a wait that one of these kernels gave up since the last check, or 0; synchronises and clears."""
        if self._branches is None:
            return 0
        L = self._branches
        codes = [L.gb_tree_attention_error_check(), L.gb_beam_select_error_check(), L.gb_branches_error_check()]
        code = next((c for c in codes if c), 0)
        if code:                # (counters that a kernel which gave up left behind are not zero)
            self._branch_scratch.clear()
        return code

    def check_branch_errors(self) -> None:
        """Synchronises, and raises if one of these kernels gave up on a wait since the last check."""
        seen, self.error_word[0] = int(self.error_word[0]), 0
        code = self.branch_error_code() or seen
        _need(not code, f"a kernel of branches gave up waiting: code {code}")

    def _here(self, *tensors):
        for t in tensors:
            _need(t.get_device() == self._device_index, "kernel operands must live on the kernel set's CUDA device")

    @staticmethod
    def _check_requests(what, cu_q, kv_lens):
        for t in (cu_q, kv_lens):
            _need(t.dtype is torch.int32 and t.is_contiguous() and t.dim() == 1, f"{what}: cu_q and kv_lens must be contiguous int32")
        R = kv_lens.shape[0]
        _need(cu_q.shape[0] == R + 1, f"{what}: cu_q has one number more than there are requests")
        return R

    # ------------------------------------------------------------------ trees
    def tree_layout(self, parents, cu_q, kv_lens, positions, mask, max_q_len: int, window: int = 0):
        """Positions and masks of a step's trees. ``parents [T]`` (int32): the token that each continues, by its number within the request
        (``cu_q[r]`` to ``cu_q[r + 1]``), or -1: the context itself; a parent comes before its children. ``kv_lens [R]``: the
        requests' lengths, their drafted tokens included. ``positions [T]`` (int32) becomes the context's length plus the number of
        ancestors, ``mask [T, words]`` (int32, 32 bits a word for at least ``max_q_len``, the longest request's tokens) a bit for the token itself and each
        ancestor; with a ``window`` w those of its last w positions. A token whose parents do not lead to -1 gets no bits
        and the context's length as position."""
        what = "tree_layout"
        i32, dev, T, R = torch.int32, self._device_index, parents.shape[0], kv_lens.shape[0]
        rows, words = mask.shape if mask.dim() == 2 else (-1, 0)
        # (one condition, taken apart when it fails)
        if not (parents.dtype is i32 and cu_q.dtype is i32 and kv_lens.dtype is i32 and positions.dtype is i32 and mask.dtype is i32 and parents.is_contiguous()
                and cu_q.is_contiguous() and kv_lens.is_contiguous() and positions.is_contiguous() and mask.is_contiguous() and parents.shape == (T,)
                and positions.shape == (T,) and rows == T and kv_lens.dim() == 1 and cu_q.shape == (R + 1,) and 0 <= max_q_len <= 32 * words <= self.MOST_DRAFTED
                and 0 <= window < 1 << 31 and parents.get_device() == dev and cu_q.get_device() == dev and kv_lens.get_device() == dev
                and positions.get_device() == dev and mask.get_device() == dev):
            self._here(parents, cu_q, kv_lens, positions, mask)
            self._check_requests(what, cu_q, kv_lens)
            for t in (parents, positions):
                _need(t.dtype is i32 and t.is_contiguous() and t.shape == (T,), f"{what}: parents and positions must be contiguous int32 [T]")
            _need(mask.dtype is i32 and mask.is_contiguous() and rows == T, f"{what}: mask must be contiguous int32 [T, words]")
            _need(0 <= max_q_len <= min(32 * words, self.MOST_DRAFTED), f"{what}: at most {self.MOST_DRAFTED} drafted tokens of a request, and 32 to a word")
            _need(32 * words <= self.MOST_DRAFTED, f"{what}: a mask of more than {self.MOST_DRAFTED} bits")
            raise KernelError(f"{what}: a window of 31 bits")
        if T == 0 or R == 0:
            return
        L = self.branch_lib
        self._check(L, L.gb_tree_layout(parents.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), positions.data_ptr(), mask.data_ptr(), words,
                                        window, R, max_q_len, self._stream()), what)

    def tree_attention(self, q, k_pool, v_pool, block_table, cu_q, kv_lens, positions, mask, out, scale, window, page_size, max_q_len, max_kv_len,
                       ws=None):
        """Grouped-query attention of drafted tokens over the paged cache: ``q [T, Hq, hd]`` and ``out [T, Hq * hd]``, pools
        ``[pages, Hkv, page_size, hd]``, all bfloat16 or all float32. Token i of request r (its tokens are ``cu_q[r]`` to ``cu_q[r + 1]``, ``kv_lens[r]`` its length
        with them) reads the request's context, with a ``window`` w > 0 only positions above ``positions[i] - w``, and those of
        the request's drafted tokens whose bits are set in ``mask[i]`` (``tree_layout`` makes both; any other mask will do, and positions from the
        context's length up to below ``kv_lens[r]``). One that reads nothing gets zeros (and so does one whose scores are all -inf). What is masked
        has no influence, whatever it holds; a value that is no finite number leaves none in its channel to those that read it, however small its weight (on the
        tensor cores it may be NaN in all channels of the head). Pages that the block table does not have (-1) count as zeros.

        On the tensor cores for bfloat16, heads of 64 and 128 and pages of 8 to 128 (a power of two), with weights rounded to bfloat16; other shapes (heads of a
        multiple of 4 channels up to 256) and float32 in 32-bit arithmetic throughout."""
        T, Hq, hd = q.shape
        pool = k_pool.shape
        pages, Hkv = pool[0], pool[1]
        table = block_table.shape
        rows, words = mask.shape
        R, dev, width = kv_lens.shape[0], self._device_index, table[1]
        dtype, i32 = q.dtype, torch.int32
        # (one condition, taken apart when it fails)
        if not (q.is_contiguous() and out.is_contiguous() and out.shape == (T, Hq * hd) and dtype is out.dtype and dtype is k_pool.dtype
                and dtype is v_pool.dtype and dtype in _TAG and pool == (pages, Hkv, page_size, hd) and v_pool.shape == pool and k_pool.is_contiguous()
                and v_pool.is_contiguous() and Hkv > 0 and Hq > 0 and Hq % Hkv == 0 and hd > 0 and block_table.dtype is i32 and cu_q.dtype is i32 and kv_lens.dtype is i32
                and positions.dtype is i32 and mask.dtype is i32 and block_table.is_contiguous() and cu_q.is_contiguous() and kv_lens.is_contiguous()
                and positions.is_contiguous() and mask.is_contiguous() and cu_q.shape == (R + 1,) and kv_lens.dim() == 1 and table[0] >= R
                and positions.shape == (T,) and rows == T and 32 * words >= max_q_len > 0 and scale > 0
                and 0 <= window < 1 << 31 and page_size > 0 and width * page_size >= max_kv_len >= 0 and max_kv_len <= self.MOST_POSITIONS
                and q.get_device() == dev and k_pool.get_device() == dev and v_pool.get_device() == dev and out.get_device() == dev
                and block_table.get_device() == dev and cu_q.get_device() == dev and kv_lens.get_device() == dev and positions.get_device() == dev and mask.get_device() == dev):
            self._refuse_attention(q, k_pool, v_pool, block_table, cu_q, kv_lens, positions, mask, out, scale, window, page_size, max_q_len,
                                   max_kv_len)
        if T == 0 or R == 0:
            return
        L, g, stream = self.branch_lib, Hq // Hkv, self._stream()
        q_ptr, k_ptr, v_ptr, out_ptr = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
        low_bits = q_ptr | k_ptr | v_ptr | out_ptr
        if (dtype is torch.bfloat16 and self.tc is not None and (hd == 64 or hd == 128) and page_size in (8, 16, 32, 64, 128) and g <= 128 and pages > 0
                and not low_bits & 15):
            # the row of all tiles, with four more for every block of rows, is counted in 31 bits
            if R * Hkv * (max_q_len * g // 64 + 1) * (max_kv_len // 128 + 6) >= 1 << 31:
                raise KernelError("tree_attention: more tiles than fit 31 bits")
            scratch, counters, _held = self._branch_memory("tree_attention", L.gb_tree_attention_scratch_bytes, (hd,), ws, stream)
            entry, launches = L.gb_tree_attention_tc, (R + 2047) // 2048
        else:
            _need(hd % 4 == 0 and hd <= 256, "tree_attention: heads of a multiple of 4 channels up to 256")
            _need(not low_bits & (15 if dtype is torch.float32 else 7), "tree_attention: operands on 16 bytes (bfloat16: 8)")
            entry, counters, scratch, launches = L.gb_tree_attention_simple, 0, 0, 1
        self._check(L, entry(_TREE_CALL.pack(
            q_ptr, k_ptr, v_ptr, out_ptr, block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), positions.data_ptr(), mask.data_ptr(), counters,
            scratch, stream, width, words, T, R, pages, Hq, Hkv, hd, window, page_size, max_q_len, max_kv_len, _TAG[dtype], scale)),
            "tree_attention", launches)

    def _refuse_attention(self, q, k_pool, v_pool, block_table, cu_q, kv_lens, positions, mask, out, scale, window, page_size, max_q_len, max_kv_len):
        what = "tree_attention"
        T, Hq, hd = q.shape
        Hkv, R = k_pool.shape[1], kv_lens.shape[0]
        shape = (k_pool.shape[0], Hkv, page_size, hd)
        self._here(q, k_pool, v_pool, out, block_table, cu_q, kv_lens, positions, mask)
        _need(q.is_contiguous() and out.is_contiguous() and out.shape == (T, Hq * hd), f"{what}: q/out shape")
        _need(q.dtype is out.dtype and q.dtype is k_pool.dtype and q.dtype is v_pool.dtype and q.dtype in _TAG,
              f"{what}: one dtype, bfloat16 or float32, for q, cache and out")
        _need(k_pool.shape == shape and v_pool.shape == shape and k_pool.is_contiguous() and v_pool.is_contiguous(),
              f"{what}: pools must be contiguous {list(shape)}")
        _need(Hkv > 0 and Hq > 0 and Hq % Hkv == 0, f"{what}: heads in whole groups")
        _need(hd > 0, f"{what}: heads of at least four channels")
        _need(page_size > 0, f"{what}: pages of at least one position")
        self._check_requests(what, cu_q, kv_lens)
        for t in (block_table, positions, mask):
            _need(t.dtype is torch.int32 and t.is_contiguous(), f"{what}: block table, positions and mask must be contiguous int32")
        _need(block_table.shape[0] >= R, f"{what}: a row of the block table for every request")
        _need(positions.shape == (T,) and mask.shape[0] == T, f"{what}: a position and a row of the mask for every token")
        _need(0 < max_q_len <= 32 * mask.shape[1], f"{what}: the mask is too narrow for that many tokens")
        _need(scale > 0 and 0 <= window < 1 << 31, f"{what}: a positive scale, a window that is not negative (and fits 31 bits)")
        _need(0 <= max_kv_len <= self.MOST_POSITIONS, f"{what}: at most {self.MOST_POSITIONS} positions of a request")
        raise KernelError(f"{what}: the block table is too narrow for that many positions")

    def tree_accept(self, tokens, targets, parents, cu_q, kv_lens, path, kept, next_tokens, max_q_len: int, pools=(), block_table=None,
                    page_size: int = 0):
        """Keeps of every request's tree what the model would have chosen itself. ``tokens``, ``targets``, ``parents`` (int32 ``[T]``): the
        drafted tokens, the token that the model chose behind each, and ``tree_layout``'s parents. From a request's token 0 on the first of the tokens that
        continue the last one and are its target is kept, until there is none. ``path [R, width]`` (int32) becomes the kept tokens' numbers, then
        -1, ``kept [R]`` how many they are (0: a request without tokens), ``next_tokens [R]`` the last one's target (-1).

        ``pools`` (each ``[calls, pages, heads, page_size, width]`` or without ``calls``; two or four bytes a number; none twice) share ``block_table``: the
        rows of kept tokens, at ``kv_lens[r]`` less the tree's size plus their numbers, go to the places right behind the context, in
        every call. Rows behind them, and where the block table has no page, are left as they are. The request's length is then its context plus
        ``kept[r]``. (A chosen token may come from any rule, a drawn one too: a token is its parent's target or is not kept.)"""
        what = "tree_accept"
        tokens_shape, i32, dev = tokens.shape, torch.int32, self._device_index
        path_shape, R = path.shape, kv_lens.shape[0]
        # (one condition, taken apart when it fails)
        if not (tokens.dtype is i32 and targets.dtype is i32 and parents.dtype is i32 and cu_q.dtype is i32 and kv_lens.dtype is i32 and path.dtype is i32
                and kept.dtype is i32 and next_tokens.dtype is i32 and tokens.is_contiguous() and targets.is_contiguous() and parents.is_contiguous()
                and cu_q.is_contiguous() and kv_lens.is_contiguous() and path.is_contiguous() and kept.is_contiguous() and next_tokens.is_contiguous()
                and len(tokens_shape) == 1 and targets.shape == tokens_shape and parents.shape == tokens_shape and cu_q.shape == (R + 1,)
                and kept.shape == (R,) and next_tokens.shape == (R,) and kv_lens.dim() == 1 and len(path_shape) == 2 and path_shape[0] == R
                and 0 < max_q_len <= self.MOST_DRAFTED and path_shape[1] >= max_q_len and R <= 65535 and tokens.get_device() == dev
                and targets.get_device() == dev and parents.get_device() == dev and cu_q.get_device() == dev and kv_lens.get_device() == dev
                and path.get_device() == dev and kept.get_device() == dev and next_tokens.get_device() == dev):
            self._here(tokens, targets, parents, cu_q, kv_lens, path, kept, next_tokens)
            self._check_requests(what, cu_q, kv_lens)
            for t in (tokens, targets, parents):
                _need(t.dtype is i32 and t.is_contiguous() and t.dim() == 1 and t.shape == tokens_shape,
                      f"{what}: tokens, targets and parents must be contiguous int32 [T]")
            for t in (kept, next_tokens):
                _need(t.dtype is i32 and t.is_contiguous() and t.shape == (R,), f"{what}: kept and next_tokens must be contiguous int32 [R]")
            _need(path.dtype is i32 and path.is_contiguous() and path.dim() == 2 and path_shape[0] == R, f"{what}: path must be contiguous int32 [R, width]")
            _need(0 < max_q_len <= self.MOST_DRAFTED, f"{what}: 1 to {self.MOST_DRAFTED} drafted tokens of a request")
            _need(path_shape[1] >= max_q_len, f"{what}: a path as wide as the largest tree")
            raise KernelError(f"{what}: at most 65,535 requests")
        pages, table, width, flat = 0, 0, 0, []
        if pools:
            if not (block_table is not None and block_table.dtype is i32 and block_table.is_contiguous() and block_table.dim() == 2
                    and block_table.get_device() == dev and block_table.shape[0] >= R):
                _need(block_table is not None, f"{what}: pools come with a block table")
                self._here(block_table)
                raise KernelError(f"{what}: the block table must be contiguous int32, a row for every request")
            table, width = block_table.data_ptr(), block_table.shape[1]
            pages = pools[0].shape[-4] if pools[0].dim() >= 4 else 0
            for pool in pools:
                shape, item = pool.shape, pool.itemsize
                if not (len(shape) in (4, 5) and pool.is_contiguous() and shape[-2] == page_size > 0 and (item == 2 or item == 4) and shape[-4] == pages
                        and pool.get_device() == dev):
                    self._here(pool)
                    _need(len(shape) in (4, 5) and pool.is_contiguous() and shape[-2] == page_size > 0,
                          f"{what}: pools must be contiguous [calls, pages, heads, page_size, width]")
                    _need(item in (2, 4), f"{what}: rows of two or four bytes a number (pages in 8 bits have a scale for all their rows)")
                    raise KernelError(f"{what}: pools of one block table have the same number of pages")
                flat += pool.data_ptr(), shape[0] if len(shape) == 5 else 1, shape[-3], shape[-1] * item
            if len({*flat[::4]}) != len(pools):
                at = [a for a in flat[::4] if a]               # (empty ones have no address)
                _need(len(set(at)) == len(at), f"{what}: a pool is given twice")
        if R == 0:
            return
        L, packed = self.branch_lib, array("q", flat)
        self._check(L, L.gb_tree_accept(_ACCEPT_CALL.pack(
            tokens.data_ptr(), targets.data_ptr(), parents.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), path.data_ptr(), kept.data_ptr(),
            next_tokens.data_ptr(), table, packed.buffer_info()[0], self._stream(), len(flat) // 4 if pages else 0, pages, path_shape[1], width, page_size, R,
            max_q_len)), what)

    # ------------------------------------------------------------------ beams
    def beam_select(self, logits, scores, best, parents, tokens, ws=None):
        """The best continuations of every item over its beams and the vocabulary: candidates (beam w, token v) have the score ``scores[i, w] +
        log_softmax(logits[i * beams + w])[v]``, with sums and what counts most in 64 bits, other exponentials in 32: off by 4e-8 as a rule, and
        where most of a row's sum are equal logits d below its largest by up to 2^-21 + 1.35e-7 d (2.1e-6 at d = 12); ``best``, ``parents``, ``tokens`` (float32, int32, int32 ``[items, n]``)
        become the n best ones' scores, beams and tokens, equal ones in the order of (w, v); beams of the same logits and score have
        equal ones, wherever their rows lie. ``logits [items * beams, V]`` float32 with rows of unit stride,
        ``scores [items, beams]`` float32. A beam whose score is not finite is over, one whose logits hold an infinity or NaN has no
        distribution: their candidates, like tokens of logit -inf, have the score -inf and come last. Up to 64 beams and 64 candidates."""
        what = "beam_select"
        items, beams = scores.shape
        (rows, V), (ld, unit) = logits.shape, logits.stride()
        n, dev, f32, i32 = best.shape[1], self._device_index, torch.float32, torch.int32
        chosen = best.shape
        if not (rows == items * beams and logits.dtype is f32 and (unit == 1 or V == 1) and scores.dtype is f32 and scores.is_contiguous()
                and best.dtype is f32 and best.is_contiguous() and parents.dtype is i32 and parents.is_contiguous() and tokens.dtype is i32
                and tokens.is_contiguous() and chosen == (items, n) and parents.shape == chosen and tokens.shape == chosen
                and 0 < n <= self.MOST_BEAMS and n <= beams * V and beams <= self.MOST_BEAMS and rows <= 65535 and V <= 1 << 30
                and logits.get_device() == dev and scores.get_device() == dev and best.get_device() == dev and parents.get_device() == dev
                and tokens.get_device() == dev):
            self._here(logits, scores, best, parents, tokens)
            _need(rows == items * beams, f"{what}: {rows} rows of logits for {items} items of {beams} beams")
            _need(logits.dtype is f32 and (unit == 1 or V == 1), f"{what}: float32 logits with rows of unit stride")
            _need(scores.dtype is f32 and scores.is_contiguous(), f"{what}: contiguous float32 scores")
            for t, dtype in ((best, f32), (parents, i32), (tokens, i32)):
                _need(t.dtype is dtype and t.is_contiguous() and t.shape == (items, n), f"{what}: best (float32), parents and tokens (int32) [items, n], contiguous")
            _need(0 < n <= min(self.MOST_BEAMS, beams * V), f"{what}: 1 to {self.MOST_BEAMS} candidates, no more than there are")
            _need(beams <= self.MOST_BEAMS, f"{what}: at most {self.MOST_BEAMS} beams")
            raise KernelError(f"{what}: at most 65,535 rows of 2^30 logits")
        if rows == 0:
            return
        L, stream = self.branch_lib, self._stream()
        scratch, counters, _held = self._branch_memory("beam_select", L.gb_beam_select_scratch_bytes, (items, beams, V, n), ws, stream)
        self._check(L, L.gb_beam_select(_BEAM_CALL.pack(
            logits.data_ptr(), scores.data_ptr(), best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), counters, scratch, stream,
            ld, items, beams, V, n)), what)

    def copy_entries(self, arrays, source, target, dim: int = 0):
        """In every one of ``arrays`` (contiguous, of any type, none of them twice): entry ``source[i]`` along ``dim`` is copied to entry
        ``target[i]``, for all i as if everything was read before anything is written: pages of pools ``[calls, pages, ...]`` with ``dim`` 1,
        states ``[slots, ...]`` with 0. ``source`` and ``target``: int32, up to 1,024. A copy with a source or target that the array does not
        have (-1) is left out; of several to one target the last one counts."""
        what = "copy_entries"
        copies, i32, dev = source.shape, torch.int32, self._device_index
        if not (source.dtype is i32 and target.dtype is i32 and source.is_contiguous() and target.is_contiguous() and len(copies) == 1
                and target.shape == copies and copies[0] <= self.MOST_COPIES and source.get_device() == dev and target.get_device() == dev):
            self._here(source, target)
            for t in (source, target):
                _need(t.dtype is i32 and t.is_contiguous() and t.dim() == 1 and t.shape == copies,
                      f"{what}: source and target must be contiguous int32 of one length")
            raise KernelError(f"{what}: {copies[0]} copies (at most {self.MOST_COPIES})")
        flat, of_shape, of_dtype = [], None, None
        for a in arrays:
            shape, dtype = a.shape, a.dtype
            if not (a.is_contiguous() and a.get_device() == dev):
                self._here(a)
                raise KernelError(f"{what}: arrays must be contiguous and have dimension {dim}")
            if shape != of_shape or dtype is not of_dtype:           # (layers' arrays are alike)
                _need(0 <= dim < len(shape), f"{what}: arrays must be contiguous and have dimension {dim}")
                of_shape, of_dtype, entries, nbytes = shape, dtype, shape[dim], a.nbytes
                outer = 1 if dim == 0 else shape[0] if dim == 1 else math.prod(shape[:dim])
            if nbytes:
                flat += a.data_ptr(), outer, entries, nbytes // (outer * entries)
        if not flat or copies[0] == 0:
            return
        L, k, packed = self.branch_lib, len(flat) // 4, array("q", flat)
        if k > 1:
            _need(len({*flat[::4]}) == k, f"{what}: an array is given twice")
        self._check(L, L.gb_copy_entries(_COPY_CALL.pack(source.data_ptr(), target.data_ptr(), packed.buffer_info()[0], self._stream(), k, copies[0])), what,
                    (k + 95) // 96)
