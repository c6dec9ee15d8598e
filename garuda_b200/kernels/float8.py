"""Weights and the paged cache in 8 bits (E4M3 with a scale per block): the checking wrappers of their kernels.

A scale is a power of two, 2^e with the smallest e >= -100 for which ``448 * 2^e`` is at least the block's largest magnitude,
so that dividing by it is exact and a value is rounded once. Blocks are 128 x 128 of a weight, 128 channels of a token, and a
page of one key/value head of the cache.
"""
from __future__ import annotations

import contextlib
import ctypes
from ctypes import c_void_p, c_int, c_float, c_longlong
from typing import NamedTuple

import torch

from ..csrc.build import load_kernel_lib
from .checks import _TAG, KernelError, _need, _tag

BLOCK = 128
E4M3 = torch.float8_e4m3fn
# (what torch.cuda.is_current_stream_capturing is, without the call around it)
_capturing = torch._C._cuda_isCurrentStreamCapturing


class Float8Weight(NamedTuple):
    """A matrix in 8 bits: ``values [N, K]`` (E4M3, rows of unit stride that start on 16 bytes) and ``scales
    [ceil(N / 128), ceil(K / 128)]`` (float32, powers of two): ``w[n, k] = values[n, k] * scales[n // 128, k // 128]``."""
    values: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.values.shape

    @property
    def dtype(self):
        return self.values.dtype

    @property
    def is_cuda(self):
        return self.values.is_cuda and self.scales.is_cuda

    def first_rows(self, n: int) -> "Float8Weight":
        """The first ``n`` rows, as a view."""
        return Float8Weight(self.values[:n], self.scales[:(n + BLOCK - 1) // BLOCK])


_FLOAT8_SIGNATURES = {
    "gb_f8_quantize_weight": [c_void_p, c_int, c_longlong, c_int, c_int, c_void_p, c_longlong, c_void_p, c_void_p],
    "gb_f8_append": [c_void_p, c_int, c_longlong, c_void_p, c_int] + [c_void_p] * 7 + [c_int] * 6 + [c_void_p, c_int, c_int, c_void_p],
    "gb_f8_attention_simple": [c_void_p, c_int] + [c_void_p] * 5 + [c_int] + [c_void_p] * 3 + [c_int] * 5 + [c_float, c_int, c_int, c_void_p],
    "gb_f8_attention_decode": [c_void_p] * 6 + [c_int] + [c_void_p] * 3 + [c_int, c_longlong] + [c_int] * 3 + [c_float] + [c_int] * 3 + [c_void_p] * 3,
    "gb_f8_attention_tile": [c_void_p] * 6 + [c_int] + [c_void_p] * 3 + [c_int, c_longlong] + [c_int] * 3 + [c_float] + [c_int] * 3 + [c_void_p],
    "gb_f8_attention_decode_rows": [c_int],
    "gb_f8_attention_tile_error_check": [],
    "gb_f8_attention_tile_set_error_sink": [c_void_p],
    "gb_f8_attention_decode_error_check": [],
    "gb_f8_attention_decode_set_error_sink": [c_void_p],
    "gb_f8_linear": [c_void_p, c_int, c_longlong, c_void_p, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_void_p,
                     c_void_p, c_void_p],
    "gb_f8_linear_plan": [c_int, c_int, c_int, c_void_p],
    "gb_f8_gemm_error_check": [],
    "gb_f8_gemm_set_error_sink": [c_void_p],
}


class Float8Ops:
    """What ``CudaOps`` has of 8 bits. Everything is launched on torch's current stream, and results do not depend on the order in which
    blocks finish.

    Scratch memory is the call's ``ws``, else that of the step that is running (``scratch_from``), else one that the set keeps for the stream, at
    the largest size that was asked for, as long as the set lives; a call that is captured into a graph without ``ws`` has memory of its
    graph's own (and clears its counters in every replay: give a captured step a ``ws`` that it ran with once). ``scratch_from`` is a
    state of the set, so a set is one thread's.

    A kernel may start while the one in front of it in the stream still runs, if that one lets it (programmatic dependent launch; the framework's
    do, torch's and copies do not). Before it waits for that one it reads what a step has from the host or from load time: lengths
    (``cu_q``, ``kv_lens``), block tables and weights. A kernel of the caller's own that lets its dependents start early must not write these
    right in front of a call; everything else may come from it."""

    #: the workspace of the step that is running (``scratch_from``): what a captured graph reads must be its own
    step_ws = None
    #: ``"float8_e4m3"``: ``hold`` keeps matrices in 8 bits
    weight_dtype = None

    @contextlib.contextmanager
    def scratch_from(self, ws):
        """Within the block, 8-bit calls that are given no workspace take their scratch memory from this one."""
        outer, self.step_ws = self.step_ws, ws
        try:
            yield
        finally:
            self.step_ws = outer

    def hold(self, w: torch.Tensor):
        """A weight matrix as this kernel set keeps it: in 8 bits if it was asked to, else as it is. ``linear`` takes both."""
        return self.float8_weight(w) if self.weight_dtype == "float8_e4m3" else w.contiguous()

    @property
    def float8_lib(self):
        """The library of the 8-bit kernels, compiled and loaded when a caller first needs it."""
        if self._float8 is None:
            L = load_kernel_lib("garuda_float8")
            L.gb_last_error.restype = ctypes.c_char_p
            for name, argtypes in _FLOAT8_SIGNATURES.items():
                fn = getattr(L, name)
                fn.argtypes, fn.restype = argtypes, c_int
            L.gb_f8_linear_scratch_bytes.argtypes = [c_int, c_int, c_int, ctypes.POINTER(c_longlong)]
            L.gb_f8_linear_scratch_bytes.restype = c_longlong
            L.gb_f8_attention_decode_part_bytes.restype = c_longlong
            self._float8_part_bytes = int(L.gb_f8_attention_decode_part_bytes())
            self._float8_sizes, self._float8_scratch, self._float8_few = {}, {}, {}
            sinks = (L.gb_f8_gemm_set_error_sink, L.gb_f8_attention_decode_set_error_sink, L.gb_f8_attention_tile_set_error_sink)
            if any([sink(self.error_word.data_ptr()) for sink in sinks]):
                _need(False, "the 8-bit library could not be given the host's error word")
            self._float8 = L
        return self._float8

    def _scratch8(self, name, nbytes, counters, counter_bytes, ws, stream):
        """Scratch bytes and counters (cleared when they are made) of these names: from the call's workspace, the running step's, or one per
        stream. A call that is captured without a workspace has memory of its graph's own, cleared in the graph: what the set keeps may
        never have been cleared, if the graph that it was made in does not run."""
        if ws is None:
            ws = self.step_ws
        if ws is None:
            if _capturing():
                return (torch.empty(nbytes, dtype=torch.uint8, device=self.device),
                        torch.zeros(counter_bytes, dtype=torch.uint8, device=self.device))
            ws = self._float8_scratch.get(stream)
            if ws is None:
                from ..engine.batch import Workspace
                ws = self._float8_scratch[stream] = Workspace(self.device)
        return ws.get(name, (nbytes,), torch.uint8), ws.get(counters, (counter_bytes,), torch.uint8, zero=True)

    def float8_error_code(self) -> int:
        """The code of a wait that an 8-bit kernel gave up since the last check, or 0; synchronises and clears."""
        if self._float8 is None:
            return 0
        L = self._float8
        codes = [L.gb_f8_gemm_error_check(), L.gb_f8_attention_decode_error_check(), L.gb_f8_attention_tile_error_check()]
        return next((c for c in codes if c), 0)

    def check_float8_errors(self) -> None:
        """Synchronises, and raises if an 8-bit kernel gave up on a wait since the last check."""
        seen, self.error_word[0] = int(self.error_word[0]), 0
        code = self.float8_error_code() or seen
        _need(not code, f"an 8-bit kernel gave up waiting: code {code}")

    # ------------------------------------------------------------------ matrix products
    def float8_weight(self, w: torch.Tensor) -> Float8Weight:
        """``w [N, K]`` (bfloat16 or float32) in 8 bits with a scale per block of 128 x 128."""
        self._on_device(w)
        _need(w.dim() == 2 and w.stride(1) == 1 and w.numel() > 0, "float8_weight: a matrix with rows of unit stride")
        N, K = w.shape
        pitch, blocks = (K + 15) // 16 * 16, ((N + BLOCK - 1) // BLOCK, (K + BLOCK - 1) // BLOCK)
        codes = torch.empty(N, pitch, dtype=E4M3, device=w.device)
        scales = torch.empty(blocks, dtype=torch.float32, device=w.device)
        self._check(self.float8_lib, self.float8_lib.gb_f8_quantize_weight(
            w.data_ptr(), _tag(w, "float8_weight"), w.stride(0), N, K, codes.data_ptr(), pitch, scales.data_ptr(), self._stream()),
            "float8_weight")
        return Float8Weight(codes[:, :K], scales)

    def linear_float8(self, a, w, out, accumulate: bool = False, alpha: float = 1.0, ws=None, gated: bool = False):
        """``out[M, N] (+)= q(a) @ w^T``: ``w`` a ``Float8Weight`` (or a pair of its two tensors), ``a [M, K]`` bfloat16 or float32, its
        rows rounded to 8 bits with a scale per token and 128 channels (``q``; an infinity counts as 448 * 2^120, next to which the rest of its
        128 channels is nothing). Sums are 32-bit; ``out`` is bfloat16 or float32, and float32 where ``accumulate`` adds ``alpha *
        product`` to what is there. A scale of the weights that is no positive power of two (``float8_weight`` makes none) turns the results
        of its 128 rows into NaN. ``gated``: ``a [M, 2 K]`` has rows ``[gate | up]``, and
        ``silu(gate) * up`` is rounded to 8 bits, from 32, and multiplied."""
        values, scales = w
        # (one condition, taken apart when it fails)
        out_tag = _TAG.get(out.dtype)
        if not (a.is_cuda and values.is_cuda and scales.is_cuda and out.is_cuda and a.dim() == 2 and values.dim() == 2 and out.dim() == 2):
            _need(a.is_cuda and values.is_cuda and scales.is_cuda and out.is_cuda, "kernel operands must live on the CUDA device")
            raise KernelError("linear_float8: operands must be matrices")
        M, width = a.shape
        N, K = values.shape
        a_row, w_row = a.stride(0), values.stride(0)
        if not (width == (2 * K if gated else K) and out.shape == (M, N) and K > 0 and values.dtype is E4M3 and scales.dtype is torch.float32
                and scales.is_contiguous() and scales.shape == ((N + 127) // 128, (K + 127) // 128) and (values.stride(1) == 1 or K == 1)
                and (w_row % 16 == 0 or N <= 1) and values.data_ptr() % 16 == 0 and (a.stride(1) == 1 or width == 1) and out_tag is not None
                and out.is_contiguous() and (out_tag == 0 if accumulate else alpha == 1.0)):
            _need(width == (2 * K if gated else K) and out.shape == (M, N),
                  f"linear_float8: shapes {tuple(a.shape)} x {tuple(values.shape)} -> {tuple(out.shape)}")
            _need(K > 0, "linear_float8: no channels")
            _need(values.dtype is E4M3, "linear_float8: weights must be float8_e4m3fn")
            _need(scales.dtype is torch.float32 and scales.is_contiguous() and scales.shape == ((N + 127) // 128, (K + 127) // 128),
                  "linear_float8: one float32 scale per block of 128 x 128")
            _need((values.stride(1) == 1 or K == 1) and (w_row % 16 == 0 or N <= 1) and values.data_ptr() % 16 == 0,
                  "linear_float8: rows of codes must start on 16 bytes (float8_weight makes such)")
            _need(a.stride(1) == 1 or width == 1, "linear_float8: rows of a must have unit stride")
            _need(out_tag is not None and out.is_contiguous(), "linear_float8: out must be contiguous, bfloat16 or float32")
            _need(not accumulate or out_tag == 0, "linear_float8: accumulates into float32 only")
            raise KernelError("linear_float8: a multiplier goes with accumulation only")
        if M == 0 or N == 0:
            return
        L, stream = self.float8_lib, self._stream()
        sizes = self._float8_sizes.get((M, N, K))
        if sizes is None:
            counter_bytes = c_longlong(0)
            scratch_bytes = int(L.gb_f8_linear_scratch_bytes(M, N, K, ctypes.byref(counter_bytes)))
            if len(self._float8_sizes) > 4096:
                self._float8_sizes.clear()
            sizes = self._float8_sizes[M, N, K] = (scratch_bytes, int(counter_bytes.value))
        scratch, counters = self._scratch8("float8_linear", sizes[0], "float8_counters", sizes[1], ws, stream)
        self._check(L, L.gb_f8_linear(a.data_ptr(), _tag(a, "linear_float8 input"), a_row, values.data_ptr(), w_row if N > 1 else (K + 15) // 16 * 16,
                                      scales.data_ptr(), out.data_ptr(), out_tag, M, N, K, accumulate, alpha, bool(gated), counters.data_ptr(),
                                      scratch.data_ptr(), stream), "linear_float8", 2)

    def linear_float8_plan(self, M: int, N: int, K: int) -> dict:
        """How ``linear_float8`` cuts a product of this shape: ``ctas`` that work on a tile together, channel ``blocks`` (of 128) to a stage,
        ``tokens`` of a tile, ``tiles``, ``workers``, ``rounds`` in which every worker has a whole tile, and how many ``share`` the rest."""
        values = (c_int * 7)()
        self._check(self.float8_lib, self.float8_lib.gb_f8_linear_plan(M, N, K, values), "linear_float8_plan", 0)
        return dict(zip(("ctas", "blocks", "tokens", "tiles", "workers", "rounds", "share"), values))

    def swiglu_float8(self, ctx, h, w_gate_up, w_down, out, accumulate: bool = False):
        """``out (+)= q(silu(g) * u) @ w_down^T`` with ``[g | u] = q(h) @ w_gate_up^T``, both weights ``Float8Weight``. Gate and up are kept
        in bfloat16 between the products: half the bytes, and 2^-9 of a number that keeps four bits behind the gate."""
        gate_up = ctx.ws.get("gate_up", (h.shape[0], w_gate_up.values.shape[0]), torch.bfloat16)
        self.linear_float8(h, w_gate_up, gate_up)
        self.linear_float8(gate_up, w_down, out, accumulate, gated=True)

    # ------------------------------------------------------------------ the cache
    @staticmethod
    def _check_cache(what, k_pool, v_pool, k_scale, v_scale, cu_q, kv_lens, block_table, kv_heads, page_size, head_dim):
        """Shapes, types and layouts of the cache and the batch; the number of requests. (One condition, taken apart when it fails.)"""
        pages, R = k_pool.shape[0], kv_lens.shape[0]
        shape, rows = (pages, kv_heads, page_size, head_dim), (pages, kv_heads)
        if (k_pool.shape == shape and v_pool.shape == shape and k_pool.dtype is E4M3 and v_pool.dtype is E4M3 and k_pool.is_contiguous()
                and v_pool.is_contiguous() and k_scale.shape == rows and v_scale.shape == rows and k_scale.dtype is torch.float32
                and v_scale.dtype is torch.float32 and k_scale.is_contiguous() and v_scale.is_contiguous()
                and cu_q.dtype is torch.int32 and kv_lens.dtype is torch.int32 and block_table.dtype is torch.int32
                and cu_q.is_contiguous() and kv_lens.is_contiguous() and block_table.is_contiguous()
                and R > 0 and cu_q.shape == (R + 1,) and block_table.dim() == 2 and block_table.shape[0] >= R
                and k_pool.is_cuda and v_pool.is_cuda and k_scale.is_cuda and v_scale.is_cuda and cu_q.is_cuda and kv_lens.is_cuda
                and block_table.is_cuda and not (k_pool.data_ptr() | v_pool.data_ptr()) & 15):
            return R
        for t in (k_pool, v_pool, k_scale, v_scale, cu_q, kv_lens, block_table):
            _need(t.is_cuda, "kernel operands must live on the CUDA device")
        for pool, scale in ((k_pool, k_scale), (v_pool, v_scale)):
            _need(pool.dtype is E4M3 and pool.is_contiguous() and pool.shape == shape and pool.data_ptr() % 16 == 0,
                  f"{what}: pools must be float8_e4m3fn {list(shape)}")
            _need(scale.dtype is torch.float32 and scale.is_contiguous() and scale.shape == rows, f"{what}: one float32 scale per page and head")
        for t in (cu_q, kv_lens, block_table):
            _need(t.dtype is torch.int32 and t.is_contiguous(), f"{what}: cu_q, kv_lens and the block table must be contiguous int32")
        raise KernelError(f"{what}: cu_q, kv_lens and the block table disagree on the number of requests")

    def kv_append_float8(self, qkv, q_out, k_pool, v_pool, k_scale, v_scale, cu_q, kv_lens, block_table, heads, kv_heads, head_dim,
                         cos_sin, interleaved, page_size):
        """Split ``qkv [T, (heads + 2 kv_heads) head_dim]`` into heads, rotate queries and keys by ``cos_sin [T, head_dim / 2, 2]``
        (``CudaOps.rope_table``; None: leave them; ``interleaved``: pairs (2i, 2i + 1) in place of (i, i + head_dim / 2)), write the
        queries to ``q_out [T, heads, head_dim]``, and keys and values in 8 bits into their pages ``[pages, kv_heads, page_size,
        head_dim]`` with one scale per page and head ``[pages, kv_heads]``. Request r's tokens ``cu_q[r]`` to ``cu_q[r + 1]`` are its last
        positions of ``kv_lens[r]``; a page that held positions before them keeps these, in its new scale where that has grown. Where the
        block table has no page (-1, or beyond its width) keys and values go nowhere."""
        what = "kv_append_float8"
        T, width = qkv.shape
        R = self._check_cache(what, k_pool, v_pool, k_scale, v_scale, cu_q, kv_lens, block_table, kv_heads, page_size, head_dim)
        _need(qkv.is_cuda and q_out.is_cuda and (cos_sin is None or cos_sin.is_cuda), "kernel operands must live on the CUDA device")
        _need(heads % kv_heads == 0 and head_dim % 16 == 0, "kv_append_float8: heads in whole groups, of a multiple of 16 channels")
        row = qkv.stride(0)
        _need(width == (heads + 2 * kv_heads) * head_dim and qkv.stride(1) == 1 and row % 2 == 0 and qkv.data_ptr() % 8 == 0,
              "kv_append_float8: qkv must be [T, (heads + 2 kv_heads) head_dim] with rows of unit stride, on 8 bytes")
        _need(q_out.is_contiguous() and q_out.shape == (T, heads, head_dim) and q_out.data_ptr() % 8 == 0, "kv_append_float8: q_out shape")
        _need(cos_sin is None or (cos_sin.dtype is torch.float32 and cos_sin.is_contiguous() and cos_sin.shape == (T, head_dim // 2, 2)
                                  and cos_sin.data_ptr() % 16 == 0), "kv_append_float8: cos_sin must be float32 [T, head_dim / 2, 2]")
        L = self.float8_lib
        self._check(L, L.gb_f8_append(
            qkv.data_ptr(), _tag(qkv, "qkv"), row, q_out.data_ptr(), _tag(q_out, "q_out"), k_pool.data_ptr(), v_pool.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(), block_table.shape[1], T, R,
            heads, kv_heads, head_dim, None if cos_sin is None else cos_sin.data_ptr(), bool(interleaved), page_size, self._stream()),
            what, 1 if T else 0)

    def paged_attention_float8(self, q, k_pool, v_pool, k_scale, v_scale, block_table, cu_q, kv_lens, out, scale, window, page_size,
                               num_requests, max_q_len, max_kv_len, ws=None, min_q_len: int = 1):
        """Causal grouped-query attention over pages of codes (``kv_append_float8``): ``q [T, Hq, hd]`` and ``out [T, Hq * hd]``
        bfloat16 (or float32, on the plain kernel). ``window`` w > 0: a query reads the last w positions, itself included. A query
        without a key to read gets zeros, one that is not finite no numbers.

        On the tensor cores (bfloat16, heads of 64 and 128, pages of 16, 32, 64 or 128) a query's channels count down to 2^-21 of its largest
        for requests of a few rows, 2^-17 for longer portions, and weights times their page's scale down to 2^-24 (2^-22 in groups of more
        than eight heads) of the row's largest. A value that is no number spoils the rows that read it and may spoil others of its request.
        Other shapes go to a kernel of one warp a row, right but up to eighty times slower."""
        what = "paged_attention_float8"
        T, Hq, hd = q.shape
        Hkv = k_pool.shape[1]
        R = self._check_cache(what, k_pool, v_pool, k_scale, v_scale, cu_q, kv_lens, block_table, Hkv, page_size, hd)
        q_ptr, out_ptr, table_width = q.data_ptr(), out.data_ptr(), block_table.shape[1]
        if not (q.is_cuda and out.is_cuda and R == num_requests and Hq % Hkv == 0 and hd % 16 == 0 and hd <= 256 and q.is_contiguous()
                and out.is_contiguous() and out.shape == (T, Hq * hd) and q.dtype is out.dtype and not (q_ptr | out_ptr) & 7 and scale > 0
                and table_width * page_size >= max_kv_len):          # (one condition, taken apart when it fails)
            _need(q.is_cuda and out.is_cuda, "kernel operands must live on the CUDA device")
            _need(R == num_requests, f"{what}: as many lengths as requests")
            _need(Hq % Hkv == 0 and hd % 16 == 0 and hd <= 256, f"{what}: heads in whole groups, of a multiple of 16 channels up to 256")
            _need(q.is_contiguous() and out.is_contiguous() and out.shape == (T, Hq * hd) and q.dtype is out.dtype, f"{what}: q/out shape")
            _need(not (q_ptr | out_ptr) & 7, f"{what}: q and out on 8 bytes")
            _need(scale > 0, f"{what}: a positive scale")
            raise KernelError(f"{what}: the block table is too narrow for that many positions")
        if T == 0:
            return
        L, g, stream = self.float8_lib, Hq // Hkv, self._stream()
        pools = (k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), table_width,
                 cu_q.data_ptr(), kv_lens.data_ptr(), out_ptr)
        if q.dtype is torch.bfloat16 and hd in (64, 128) and page_size in (16, 32, 64, 128) and g <= 128 and not (q_ptr | out_ptr) & 15:
            # requests of a few rows (new tokens times heads of a group) go to one kernel, the others to the other; groups of more than
            # sixteen heads have none of a few (a request without tokens is nobody's)
            few = self._float8_few.get(g)
            if few is None:
                few = self._float8_few[g] = L.gb_f8_attention_decode_rows(g)
            if few and min_q_len * g <= few:
                scratch, counters = self._scratch8("float8_attention_parts", self._float8_part_bytes, "float8_attention_counters", 4 * R * Hkv, ws,
                                                   stream)
                self._check(L, L.gb_f8_attention_decode(
                    q_ptr, *pools, R, k_pool.shape[0], Hq, Hkv, hd, scale, window, page_size, max_kv_len, scratch.data_ptr(),
                    counters.data_ptr(), stream), what)
            if max_q_len * g > few:
                self._check(L, L.gb_f8_attention_tile(q_ptr, *pools, R, k_pool.shape[0], Hq, Hkv, hd, scale, window, page_size, max_q_len, stream),
                            what)
            return
        self._check(L, L.gb_f8_attention_simple(q_ptr, _tag(q, "attention q"), *pools, T, R, Hq, Hkv, hd, scale, window, page_size, stream), what)
