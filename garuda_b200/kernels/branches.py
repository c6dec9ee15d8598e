"""Decoding along several branches: the checking wrappers of its kernels.

A step may bring a *tree* of drafted tokens per request instead of a stretch: token 0 is the request's last one, which the cache does not hold
yet, and ``parents`` names for every other the token of the same request that it continues. The tokens' keys and values are in the cache,
behind the request's context in the order of the tokens' numbers (``rope_kv_append`` with those places as positions and the rotation's table
made from ``tree_layout``'s). A step with trees goes: ``tree_layout`` once, ``tree_attention`` in every layer, and behind the logits
``tree_accept``, which keeps the tokens that the model would have chosen itself and moves what they left in the cache together.

*Beams* are requests of their own over shared pages: ``beam_select`` chooses how they go on, ``copy_entries`` gives a beam that goes on in several
ways a copy of its last page and of its states (``PagedCache.fork`` says which).
"""
from __future__ import annotations

import ctypes
from ctypes import c_void_p, c_int, c_float, c_longlong

import torch

from ..csrc.build import load_kernel_lib
from .checks import _TAG, KernelError, _need

_capturing = torch._C._cuda_isCurrentStreamCapturing

_SIGNATURES = {
    "gb_tree_layout": [c_void_p] * 5 + [c_int] * 4 + [c_void_p],
    "gb_tree_accept": [c_void_p] * 6 + [c_int] + [c_void_p] * 2 + [c_int] + [c_void_p] * 4 + [c_longlong, c_void_p] + [c_int] * 4 + [c_void_p],
    "gb_tree_attention_tc": [c_void_p] * 4 + [c_int] + [c_void_p] * 4 + [c_int, c_void_p, c_int, c_int, c_longlong] + [c_int] * 3 + [c_float]
    + [c_int] * 4 + [c_void_p] * 3,
    "gb_tree_attention_simple": [c_void_p, c_int] + [c_void_p] * 3 + [c_int] + [c_void_p] * 4 + [c_int, c_void_p, c_int, c_int, c_longlong]
    + [c_int] * 3 + [c_float] + [c_int] * 4 + [c_void_p],
    "gb_beam_select": [c_void_p, c_longlong, c_void_p] + [c_int] * 4 + [c_void_p] * 6,
    "gb_copy_entries": [c_int] + [c_void_p] * 6 + [c_int, c_void_p],
    "gb_tree_attention_error_check": [],
    "gb_tree_attention_set_error_sink": [c_void_p],
    "gb_beam_select_error_check": [],
    "gb_beam_select_set_error_sink": [c_void_p],
    "gb_branches_error_check": [],
    "gb_branches_set_error_sink": [c_void_p],
}


class BranchOps:
    """What ``CudaOps`` has of branches. Everything is launched on torch's current stream; results do not depend on the order in which blocks
    finish. Scratch memory is the call's ``ws``, else that of the step that is running (``scratch_from``), else one that the set
    keeps for the stream; a call captured into a graph without ``ws`` has memory of its graph's own. One ``ws`` is for one stream at a time."""

    #: ``tree_layout`` and ``tree_accept`` take trees of up to this many tokens
    MOST_DRAFTED = 8192
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
        """Scratch and counters (zero when they are made) of a call; ``sizes`` is the library's function that gives their bytes."""
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
        if ws is None:
            if _capturing():
                return (torch.empty(nbytes, dtype=torch.uint8, device=self.device),
                        torch.zeros(counter_bytes, dtype=torch.uint8, device=self.device))
            ws = self._branch_scratch.get(stream)
            if ws is None:
                from ..engine.batch import Workspace
                ws = self._branch_scratch[stream] = Workspace(self.device)
        return ws.get(name, (nbytes,), torch.uint8), ws.get(name + "_counters", (counter_bytes,), torch.uint8, zero=True)

    def branch_error_code(self) -> int:
        """The code of a wait that one of these kernels gave up since the last check, or 0; synchronises and clears."""
        if self._branches is None:
            return 0
        L = self._branches
        codes = [L.gb_tree_attention_error_check(), L.gb_beam_select_error_check(), L.gb_branches_error_check()]
        return next((c for c in codes if c), 0)

    def check_branch_errors(self) -> None:
        """Synchronises, and raises if one of these kernels gave up on a wait since the last check."""
        seen, self.error_word[0] = int(self.error_word[0]), 0
        code = self.branch_error_code() or seen
        _need(not code, f"a kernel of branches gave up waiting: code {code}")

    def _here(self, *tensors):
        for t in tensors:
            _need(t.get_device() == self._device_index, "kernel operands must live on the kernel set's CUDA device")

    @staticmethod
    def _check_requests(what, T, cu_q, kv_lens):
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
        self._here(parents, cu_q, kv_lens, positions, mask)
        T = parents.shape[0]
        R = self._check_requests(what, T, cu_q, kv_lens)
        for t in (parents, positions):
            _need(t.dtype is torch.int32 and t.is_contiguous() and t.shape == (T,), f"{what}: parents and positions must be contiguous int32 [T]")
        _need(mask.dtype is torch.int32 and mask.is_contiguous() and mask.dim() == 2 and mask.shape[0] == T, f"{what}: mask must be contiguous int32 [T, words]")
        _need(0 <= max_q_len <= min(32 * mask.shape[1], self.MOST_DRAFTED), f"{what}: at most {self.MOST_DRAFTED} drafted tokens of a request, and 32 to a word")
        _need(mask.shape[1] * 32 <= self.MOST_DRAFTED, f"{what}: a mask of more than {self.MOST_DRAFTED} bits")
        _need(window >= 0, f"{what}: a window cannot be negative")
        if T == 0 or R == 0:
            return
        L = self.branch_lib
        self._check(L, L.gb_tree_layout(parents.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), positions.data_ptr(), mask.data_ptr(), mask.shape[1],
                                        window, R, max_q_len, self._stream()), what)

    def tree_attention(self, q, k_pool, v_pool, block_table, cu_q, kv_lens, positions, mask, out, scale, window, page_size, max_q_len, max_kv_len,
                       ws=None):
        """Grouped-query attention of drafted tokens over the paged cache: ``q [T, Hq, hd]`` and ``out [T, Hq * hd]``, pools
        ``[pages, Hkv, page_size, hd]``, all bfloat16 or all float32. Token i of request r (its tokens are ``cu_q[r]`` to ``cu_q[r + 1]``, ``kv_lens[r]`` its length
        with them) reads the request's context, with a ``window`` w > 0 only positions above ``positions[i] - w``, and those of
        the request's drafted tokens whose bits are set in ``mask[i]`` (``tree_layout`` makes both; any other mask will do, and positions from the
        context's length up to below ``kv_lens[r]``). One that reads nothing gets zeros. What is masked has no influence, whatever it holds; a
        value that is no finite number makes those that read it no numbers (float32: in its channel). Pages that the block table does not
        have (-1) count as zeros.

        On the tensor cores for bfloat16, heads of 64 and 128 and pages of 8 to 128 (a power of two), with weights rounded to bfloat16; other shapes (heads of a
        multiple of 4 channels up to 256) and float32 in 32-bit arithmetic throughout."""
        what = "tree_attention"
        T, Hq, hd = q.shape
        pages, Hkv = k_pool.shape[0], k_pool.shape[1]
        R, dev, width, words = kv_lens.shape[0], self._device_index, block_table.shape[1], mask.shape[1]
        dtype, i32 = q.dtype, torch.int32
        shape = (pages, Hkv, page_size, hd)
        # (one condition, taken apart when it fails)
        if not (q.is_contiguous() and out.is_contiguous() and out.shape == (T, Hq * hd) and dtype is out.dtype and dtype is k_pool.dtype
                and dtype is v_pool.dtype and dtype in _TAG and k_pool.shape == shape and v_pool.shape == shape and k_pool.is_contiguous()
                and v_pool.is_contiguous() and Hkv > 0 and Hq % Hkv == 0 and block_table.dtype is i32 and cu_q.dtype is i32 and kv_lens.dtype is i32
                and positions.dtype is i32 and mask.dtype is i32 and block_table.is_contiguous() and cu_q.is_contiguous() and kv_lens.is_contiguous()
                and positions.is_contiguous() and mask.is_contiguous() and cu_q.shape == (R + 1,) and kv_lens.dim() == 1 and block_table.shape[0] >= R
                and positions.shape == (T,) and mask.shape[0] == T and 32 * words >= max_q_len and max_q_len > 0 and scale > 0 and window >= 0
                and width * page_size >= max_kv_len and q.get_device() == dev and k_pool.get_device() == dev and v_pool.get_device() == dev
                and out.get_device() == dev and block_table.get_device() == dev and cu_q.get_device() == dev and kv_lens.get_device() == dev
                and positions.get_device() == dev and mask.get_device() == dev):
            self._here(q, k_pool, v_pool, out, block_table, cu_q, kv_lens, positions, mask)
            _need(q.is_contiguous() and out.is_contiguous() and out.shape == (T, Hq * hd), f"{what}: q/out shape")
            _need(dtype is out.dtype and dtype is k_pool.dtype and dtype is v_pool.dtype and dtype in _TAG,
                  f"{what}: one dtype, bfloat16 or float32, for q, cache and out")
            _need(k_pool.shape == shape and v_pool.shape == shape and k_pool.is_contiguous() and v_pool.is_contiguous(),
                  f"{what}: pools must be contiguous {list(shape)}")
            _need(Hkv > 0 and Hq % Hkv == 0, f"{what}: heads in whole groups")
            self._check_requests(what, T, cu_q, kv_lens)
            for t in (block_table, positions, mask):
                _need(t.dtype is i32 and t.is_contiguous(), f"{what}: block table, positions and mask must be contiguous int32")
            _need(block_table.shape[0] >= R, f"{what}: a row of the block table for every request")
            _need(positions.shape == (T,) and mask.shape[0] == T, f"{what}: a position and a row of the mask for every token")
            _need(max_q_len > 0 and 32 * words >= max_q_len, f"{what}: the mask is too narrow for that many tokens")
            _need(scale > 0 and window >= 0, f"{what}: a positive scale, a window that is not negative")
            raise KernelError(f"{what}: the block table is too narrow for that many positions")
        if T == 0 or R == 0:
            return
        L, g, stream = self.branch_lib, Hq // Hkv, self._stream()
        q_ptr, k_ptr, v_ptr, out_ptr = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
        if (dtype is torch.bfloat16 and self.tc is not None and (hd == 64 or hd == 128) and page_size in (8, 16, 32, 64, 128) and g <= 128 and pages > 0
                and not (q_ptr | k_ptr | v_ptr | out_ptr) & 15):
            # the row of all tiles is counted in 31 bits
            _need(R * Hkv * (max_q_len * g // 64 + 1) * (max_kv_len // 128 + 2) < 1 << 31, f"{what}: more tiles than fit 31 bits")
            scratch, counters = self._branch_memory("tree_attention", L.gb_tree_attention_scratch_bytes, (hd,), ws, stream)
            self._check(L, L.gb_tree_attention_tc(q_ptr, k_ptr, v_ptr, block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(),
                                                  positions.data_ptr(), mask.data_ptr(), words, out_ptr, T, R, pages, Hq, Hkv, hd, scale, window,
                                                  page_size, max_q_len, max_kv_len, counters.data_ptr(), scratch.data_ptr(), stream), what,
                        (R + 2047) // 2048)
            return
        _need(hd % 4 == 0 and hd <= 256, f"{what}: heads of a multiple of 4 channels up to 256")
        _need(not (q_ptr | k_ptr | v_ptr | out_ptr) & (15 if dtype is torch.float32 else 7), f"{what}: operands on 16 bytes (bfloat16: 8)")
        self._check(L, L.gb_tree_attention_simple(q_ptr, _TAG[dtype], k_ptr, v_ptr, block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(),
                                                  positions.data_ptr(), mask.data_ptr(), words, out_ptr, T, R, pages, Hq, Hkv, hd, scale, window,
                                                  page_size, max_q_len, max_kv_len, stream), what)

    def tree_accept(self, tokens, targets, parents, cu_q, kv_lens, path, kept, next_tokens, max_q_len: int, pools=(), block_table=None,
                    page_size: int = 0):
        """Keeps of every request's tree what the model would have chosen itself. ``tokens``, ``targets``, ``parents`` (int32 ``[T]``): the
        drafted tokens, the token that the model chose behind each, and ``tree_layout``'s parents. From a request's token 0 on the first of the tokens that
        continue the last one and are its target is kept, until there is none. ``path [R, width]`` (int32) becomes the kept tokens' numbers, then
        -1, ``kept [R]`` how many they are (0: a request without tokens), ``next_tokens [R]`` the last one's target (-1).

        ``pools`` (each ``[calls, pages, heads, page_size, width]`` or without ``calls``; two or four bytes a number) share ``block_table``: the
        rows of kept tokens, at ``kv_lens[r]`` less the tree's size plus their numbers, go to the places right behind the context, in
        every call. Rows behind them, and where the block table has no page, are left as they are. The request's length is then its context plus
        ``kept[r]``. (A chosen token may come from any rule, a drawn one too: a token is its parent's target or is not kept.)"""
        what = "tree_accept"
        T = tokens.shape[0]
        self._here(tokens, targets, parents, cu_q, kv_lens, path, kept, next_tokens)
        R = self._check_requests(what, T, cu_q, kv_lens)
        for t in (tokens, targets, parents):
            _need(t.dtype is torch.int32 and t.is_contiguous() and t.shape == (T,), f"{what}: tokens, targets and parents must be contiguous int32 [T]")
        for t in (kept, next_tokens):
            _need(t.dtype is torch.int32 and t.is_contiguous() and t.shape == (R,), f"{what}: kept and next_tokens must be contiguous int32 [R]")
        _need(path.dtype is torch.int32 and path.is_contiguous() and path.dim() == 2 and path.shape[0] == R, f"{what}: path must be contiguous int32 [R, width]")
        _need(0 < max_q_len <= self.MOST_DRAFTED, f"{what}: 1 to {self.MOST_DRAFTED} drafted tokens of a request")
        _need(path.shape[1] >= max_q_len, f"{what}: a path as wide as the largest tree")
        _need(R <= 65535, f"{what}: at most 65,535 requests")
        n, pages, table, width = len(pools), 0, None, 0
        at, calls, heads, rows = [], [], [], []
        if n:
            _need(block_table is not None, f"{what}: pools come with a block table")
            self._here(block_table, *pools)
            _need(block_table.dtype is torch.int32 and block_table.is_contiguous() and block_table.dim() == 2 and block_table.shape[0] >= R,
                  f"{what}: the block table must be contiguous int32, a row for every request")
            table, width = block_table.data_ptr(), block_table.shape[1]
            for pool in pools:
                shape = tuple(pool.shape) if pool.dim() == 5 else (1,) + tuple(pool.shape)
                _need(len(shape) == 5 and pool.is_contiguous() and shape[3] == page_size and page_size > 0,
                      f"{what}: pools must be contiguous [calls, pages, heads, page_size, width]")
                _need(pool.dtype.itemsize in (2, 4), f"{what}: rows of two or four bytes a number (pages in 8 bits have a scale for all their rows)")
                _need(not at or shape[1] == pages, f"{what}: pools of one block table have the same number of pages")
                pages = shape[1]
                if pool.numel():
                    at.append(pool.data_ptr())
                    calls.append(shape[0])
                    heads.append(shape[2])
                    rows.append(shape[4] * pool.dtype.itemsize)
            n = len(at)
        if R == 0:
            return
        L, ints = self.branch_lib, c_int * max(n, 1)
        self._check(L, L.gb_tree_accept(tokens.data_ptr(), targets.data_ptr(), parents.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), path.data_ptr(),
                                        path.shape[1], kept.data_ptr(), next_tokens.data_ptr(), n, (c_void_p * max(n, 1))(*at), ints(*calls), ints(*heads),
                                        ints(*rows), pages, table, width, page_size, R, max_q_len, self._stream()), what)

    # ------------------------------------------------------------------ beams
    def beam_select(self, logits, scores, best, parents, tokens, ws=None):
        """The best continuations of every item over its beams and the vocabulary: candidates (beam w, token v) have the score ``scores[i, w] +
        log_softmax(logits[i * beams + w])[v]``, computed in 64 bits; ``best``, ``parents``, ``tokens`` (float32, int32, int32 ``[items, n]``)
        become the n best ones' scores, beams and tokens, equal ones in the order of (w, v). ``logits [items * beams, V]`` float32 with rows of unit stride,
        ``scores [items, beams]`` float32. A beam whose score is not finite is over, one whose logits hold an infinity or NaN has no
        distribution: their candidates, like tokens of logit -inf, have the score -inf and come last. Up to 64 beams and 64 candidates."""
        what = "beam_select"
        items, beams = scores.shape
        rows, V = logits.shape
        n, dev, f32, i32 = best.shape[1], self._device_index, torch.float32, torch.int32
        if not (rows == items * beams and logits.dtype is f32 and (logits.stride(1) == 1 or V == 1) and scores.dtype is f32 and scores.is_contiguous()
                and best.dtype is f32 and best.is_contiguous() and parents.dtype is i32 and parents.is_contiguous() and tokens.dtype is i32
                and tokens.is_contiguous() and best.shape == (items, n) and parents.shape == best.shape and tokens.shape == best.shape
                and 0 < n <= min(self.MOST_BEAMS, beams * V) and beams <= self.MOST_BEAMS and rows <= 65535 and V <= 1 << 30
                and logits.get_device() == dev and scores.get_device() == dev and best.get_device() == dev and parents.get_device() == dev
                and tokens.get_device() == dev):
            self._here(logits, scores, best, parents, tokens)
            _need(rows == items * beams, f"{what}: {rows} rows of logits for {items} items of {beams} beams")
            _need(logits.dtype is f32 and (logits.stride(1) == 1 or V == 1), f"{what}: float32 logits with rows of unit stride")
            _need(scores.dtype is f32 and scores.is_contiguous(), f"{what}: contiguous float32 scores")
            for t, dtype in ((best, f32), (parents, i32), (tokens, i32)):
                _need(t.dtype is dtype and t.is_contiguous() and t.shape == (items, n), f"{what}: best (float32), parents and tokens (int32) [items, n], contiguous")
            _need(0 < n <= min(self.MOST_BEAMS, beams * V), f"{what}: 1 to {self.MOST_BEAMS} candidates, no more than there are")
            _need(beams <= self.MOST_BEAMS, f"{what}: at most {self.MOST_BEAMS} beams")
            raise KernelError(f"{what}: at most 65,535 rows of 2^30 logits")
        if rows == 0:
            return
        L, stream = self.branch_lib, self._stream()
        scratch, counters = self._branch_memory("beam_select", L.gb_beam_select_scratch_bytes, (items, beams, V, n), ws, stream)
        self._check(L, L.gb_beam_select(logits.data_ptr(), logits.stride(0), scores.data_ptr(), items, beams, V, n, best.data_ptr(), parents.data_ptr(),
                                        tokens.data_ptr(), counters.data_ptr(), scratch.data_ptr(), stream), what)

    def copy_entries(self, arrays, source, target, dim: int = 0):
        """In every one of ``arrays`` (contiguous, of any type, none of them twice): entry ``source[i]`` along ``dim`` is copied to entry
        ``target[i]``, for all i as if everything was read before anything is written: pages of pools ``[calls, pages, ...]`` with ``dim`` 1,
        states ``[slots, ...]`` with 0. ``source`` and ``target``: int32, up to 1,024. A copy with a source or target that the array does not
        have (-1) is left out; of several to one target the last one counts."""
        what = "copy_entries"
        self._here(source, target, *arrays)
        n = source.shape[0]
        for t in (source, target):
            _need(t.dtype is torch.int32 and t.is_contiguous() and t.shape == (n,), f"{what}: source and target must be contiguous int32 of one length")
        _need(n <= self.MOST_COPIES, f"{what}: {n} copies (at most {self.MOST_COPIES})")
        at, outer, entries, nbytes = [], [], [], []
        for a in arrays:
            _need(a.is_contiguous() and 0 <= dim < a.dim(), f"{what}: arrays must be contiguous and have dimension {dim}")
            size, count = a.numel() * a.dtype.itemsize, a.shape[dim]
            if size:
                above = 1
                for d in a.shape[:dim]:
                    above *= d
                at.append(a.data_ptr())
                outer.append(above)
                entries.append(count)
                nbytes.append(size // (above * count))
        if n == 0 or not at:
            return
        k = len(at)
        L, ints = self.branch_lib, c_int * k
        self._check(L, L.gb_copy_entries(k, (c_void_p * k)(*at), ints(*outer), ints(*entries), (c_longlong * k)(*nbytes), source.data_ptr(),
                                         target.data_ptr(), n, self._stream()), what, (k + 95) // 96)
