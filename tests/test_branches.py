"""Decoding along branches, what needs no GPU: what the wrappers refuse and what they hand on."""
import ctypes
import struct
import types

import pytest
import torch

from garuda_b200.engine.batch import Workspace
from garuda_b200.kernels.branches import BranchOps
from garuda_b200.kernels.checks import KernelError

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class Recorder(BranchOps):
    """The wrappers over a library that only notes its calls; CPU tensors count as the device's (their device has the number -1)."""
    _device_index, step_ws, tc, device = -1, Workspace(torch.device("cpu")), object(), torch.device("cpu")

    def __init__(self):
        self.calls, self.launches = [], 0
        self._branch_sizes, self._branch_scratch = {}, {}

        def entry(name):
            def call(*args):
                self.calls.append((name, args))
                if name == "gb_copy_entries":          # (what it points to lives as long as the call)
                    at, n = struct.unpack("=4Q2q", args[0])[2], struct.unpack("=4Q2q", args[0])[4]
                    self.arrays = [list((ctypes.c_longlong * 4).from_address(at + 32 * i))[1:] for i in range(n)]
                return 0
            return call

        self._branches = types.SimpleNamespace(**{n: entry(n) for n in (
            "gb_tree_layout", "gb_tree_accept", "gb_tree_attention_tc", "gb_tree_attention_simple", "gb_beam_select", "gb_copy_entries",
            "gb_tree_attention_scratch_bytes", "gb_beam_select_scratch_bytes")})

    def _stream(self):
        return 0

    def _check(self, lib, code, what, kernels=1):
        self.launches += kernels

    def names(self):
        return [n for n, _ in self.calls if not n.endswith("_bytes")]


def zeros(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def attention_args(**change):
    T, R, heads, kv_heads, hd, page, dtype = 5, 2, 8, 2, change.pop("hd", 64), change.pop("page", 32), change.pop("dtype", BF16)
    args = dict(q=zeros(T, heads, hd, dtype=dtype), k_pool=zeros(4, kv_heads, page, hd, dtype=dtype), v_pool=zeros(4, kv_heads, page, hd, dtype=dtype),
                block_table=zeros(R, 2), cu_q=zeros(R + 1), kv_lens=zeros(R), positions=zeros(T), mask=zeros(T, 1), out=zeros(T, heads * hd, dtype=dtype),
                scale=0.1, window=0, page_size=page, max_q_len=3, max_kv_len=2 * page)
    return dict(args, **change)


@pytest.mark.parametrize("change, kernel", [({}, "gb_tree_attention_tc"), ({"hd": 128, "page": 8}, "gb_tree_attention_tc"), ({"hd": 48}, "gb_tree_attention_simple"),
                                            ({"page": 24}, "gb_tree_attention_simple"), ({"dtype": F32}, "gb_tree_attention_simple"),
                                            ({"page": 256}, "gb_tree_attention_simple")])
def test_attention_goes_to(change, kernel):
    ops = Recorder()
    ops.tree_attention(**attention_args(**change))
    assert ops.names() == [kernel] and ops.launches == 1


@pytest.mark.parametrize("change, match", [
    ({"q": zeros(5, 8, 64, dtype=F32)}, "one dtype"), ({"q": zeros(5, 64, 8, dtype=BF16).transpose(1, 2)}, "q/out shape"), ({"out": zeros(4, 512, dtype=BF16)}, "q/out shape"),
    ({"k_pool": zeros(4, 2, 16, 64, dtype=BF16)}, "pools"), ({"v_pool": zeros(4, 2, 32, 32, dtype=BF16)}, "pools"), ({"k_pool": zeros(4, 3, 32, 64, dtype=BF16),
      "v_pool": zeros(4, 3, 32, 64, dtype=BF16)}, "whole groups"), ({"cu_q": zeros(2)}, "cu_q"), ({"kv_lens": torch.zeros(2)}, "cu_q and kv_lens"),
    ({"block_table": zeros(1, 2)}, "a row of the block table"), ({"block_table": zeros(2, 4)[:, ::2]}, "contiguous int32"), ({"mask": zeros(4, 1)}, "a row of the mask"),
    ({"mask": zeros(5, 1, dtype=torch.int64)}, "contiguous int32"), ({"positions": zeros(4)}, "a position"), ({"max_q_len": 33}, "too narrow for that many tokens"),
    ({"scale": -1.0}, "positive scale"), ({"window": -1}, "not negative"), ({"max_kv_len": 65}, "too narrow for that many positions"),
    ({"hd": 66}, "multiple of 4"), ({"hd": 260, "dtype": F32}, "up to 256")])
def test_attention_refuses(change, match):
    ops = Recorder()
    with pytest.raises(KernelError, match=match):
        ops.tree_attention(**attention_args(**change))
    assert not ops.names()


def test_attention_of_nothing_launches_nothing():
    ops = Recorder()
    ops.tree_attention(**attention_args(q=zeros(0, 8, 64, dtype=BF16), out=zeros(0, 512, dtype=BF16), positions=zeros(0), mask=zeros(0, 1)))
    assert not ops.calls


def test_other_devices_are_refused():
    ops = Recorder()
    ops._device_index = 0
    for call in (lambda: ops.tree_attention(**attention_args()), lambda: ops.tree_layout(zeros(3), zeros(2), zeros(1), zeros(3), zeros(3, 1), 3),
                 lambda: ops.beam_select(zeros(2, 9, dtype=F32), zeros(1, 2, dtype=F32), zeros(1, 3, dtype=F32), zeros(1, 3), zeros(1, 3)),
                 lambda: ops.copy_entries([zeros(3, 3)], zeros(1), zeros(1)),
                 lambda: ops.tree_accept(zeros(3), zeros(3), zeros(3), zeros(2), zeros(1), zeros(1, 3), zeros(1), zeros(1), 3)):
        with pytest.raises(KernelError, match="device"):
            call()


@pytest.mark.parametrize("change, match", [
    ({"parents": zeros(5, dtype=torch.int64)}, "parents and positions"), ({"positions": zeros(4)}, "parents and positions"), ({"mask": zeros(4, 1)}, "mask must be"),
    ({"cu_q": zeros(4)}, "cu_q"), ({"max_q_len": 33}, "32 to a word"), ({"window": -2}, "window"), ({"mask": zeros(5, 300), "max_q_len": 9000}, "at most 8192")])
def test_layout_refuses(change, match):
    ops = Recorder()
    args = dict(dict(parents=zeros(5), cu_q=zeros(3), kv_lens=zeros(2), positions=zeros(5), mask=zeros(5, 1), max_q_len=3), **change)
    with pytest.raises(KernelError, match=match):
        ops.tree_layout(**args)
    assert not ops.names()


@pytest.mark.parametrize("change, match", [
    ({"tokens": zeros(5, dtype=torch.int64)}, "tokens, targets"), ({"targets": zeros(4)}, "tokens, targets"), ({"kept": zeros(3)}, "kept and next"), ({"path": zeros(2, 2)}, "as wide"),
    ({"path": zeros(3, 4)}, "path must be"), ({"max_q_len": 0}, "drafted tokens"), ({"block_table": None}, "come with a block table"), ({"page_size": 16}, "pools must be"),
    ({"pools": [zeros(2, 4, 2, 32, 64, dtype=torch.float8_e4m3fn)]}, "8 bits"), ({"pools": [zeros(2, 4, 2, 32, 64), zeros(2, 5, 2, 32, 64)]}, "same number of pages"),
    ({"pools": [zeros(2, 4, 2, 64, 32).transpose(3, 4)]}, "pools must be"), ({"block_table": zeros(1, 3)}, "block table must be")])
def test_accept_refuses(change, match):
    ops = Recorder()
    args = dict(dict(tokens=zeros(5), targets=zeros(5), parents=zeros(5), cu_q=zeros(3), kv_lens=zeros(2), path=zeros(2, 3), kept=zeros(2), next_tokens=zeros(2),
                     max_q_len=3, pools=[zeros(2, 4, 2, 32, 64, dtype=BF16)], block_table=zeros(2, 3), page_size=32), **change)
    with pytest.raises(KernelError, match=match):
        ops.tree_accept(**args)
    assert not ops.names()


@pytest.mark.parametrize("change, match", [
    ({"logits": zeros(5, 9, dtype=F32)}, "rows of logits"), ({"logits": zeros(6, 9, dtype=BF16)}, "float32 logits"), ({"logits": zeros(9, 6, dtype=F32).t()}, "unit stride"),
    ({"scores": zeros(2, 3, dtype=torch.float64)}, "float32 scores"), ({"best": zeros(2, 5, dtype=F32)}, "best"), ({"parents": zeros(2, 4, dtype=torch.int64)}, "best"),
    ({"best": zeros(2, 28, dtype=F32), "parents": zeros(2, 28), "tokens": zeros(2, 28)}, "no more than there are"),
    ({"best": zeros(2, 0, dtype=F32), "parents": zeros(2, 0), "tokens": zeros(2, 0)}, "1 to 64")])
def test_beam_refuses(change, match):
    ops = Recorder()
    args = dict(dict(logits=zeros(6, 9, dtype=F32), scores=zeros(2, 3, dtype=F32), best=zeros(2, 4, dtype=F32), parents=zeros(2, 4), tokens=zeros(2, 4)), **change)
    with pytest.raises(KernelError, match=match):
        ops.beam_select(**args)
    assert not ops.names()


def test_more_beams_than_there_is_room_for_are_refused():
    ops = Recorder()
    with pytest.raises(KernelError, match="at most 64 beams"):
        ops.beam_select(zeros(65, 9, dtype=F32), zeros(1, 65, dtype=F32), zeros(1, 4, dtype=F32), zeros(1, 4), zeros(1, 4))


@pytest.mark.parametrize("change, match", [
    ({"source": zeros(2)}, "one length"), ({"target": zeros(3, dtype=torch.int64)}, "contiguous int32"), ({"arrays": [zeros(4, 6).t()]}, "contiguous"),
    ({"dim": 2}, "dimension 2"), ({"source": zeros(1025), "target": zeros(1025)}, "at most 1024")])
def test_copies_refuse(change, match):
    ops = Recorder()
    args = dict(dict(arrays=[zeros(4, 6)], source=zeros(3), target=zeros(3), dim=1), **change)
    with pytest.raises(KernelError, match=match):
        ops.copy_entries(**args)
    assert not ops.names()


def test_copies_hand_on_shapes_and_leave_out_empty_arrays():
    ops = Recorder()
    ops.copy_entries([zeros(3, 7, 2, 4), zeros(3, 0, 2), zeros(2, 5, dtype=torch.uint8)], zeros(2), zeros(2), 1)
    (name, (packed,)), = ops.calls
    assert name == "gb_copy_entries" and struct.unpack("=4Q2q", packed)[4:] == (2, 2)
    assert ops.arrays == [[3, 7, 32], [2, 5, 1]]
    ops.copy_entries([zeros(3, 7)], zeros(0), zeros(0))
    ops.copy_entries([], zeros(2), zeros(2))
    assert len(ops.calls) == 1


def test_what_would_not_fit_the_kernels_numbers_is_refused():
    ops = Recorder()
    for window in (1 << 31, (1 << 32) + 5):
        with pytest.raises(KernelError, match="31 bits"):
            ops.tree_attention(**attention_args(window=window))
        with pytest.raises(KernelError, match="31 bits"):
            ops.tree_layout(zeros(5), zeros(3), zeros(2), zeros(5), zeros(5, 1), 3, window)
    wide = zeros(2, ((1 << 30) + 128) // 128)
    with pytest.raises(KernelError, match="positions of a request"):
        ops.tree_attention(**attention_args(page=128, block_table=wide, max_kv_len=(1 << 30) + 1))
    assert not ops.names()
    ops.tree_attention(**attention_args(page=128, block_table=wide, max_kv_len=1 << 30, window=(1 << 31) - 1))
    assert len(ops.names()) == 1


def test_an_array_given_twice_is_refused():
    ops = Recorder()
    pool, empty = zeros(2, 4, 2, 32, 64, dtype=BF16), zeros(0, 4, 2, 32, 64, dtype=BF16)
    accept = dict(tokens=zeros(5), targets=zeros(5), parents=zeros(5), cu_q=zeros(3), kv_lens=zeros(2), path=zeros(2, 3), kept=zeros(2), next_tokens=zeros(2),
                  max_q_len=3, block_table=zeros(2, 3), page_size=32)
    with pytest.raises(KernelError, match="given twice"):
        ops.tree_accept(pools=[pool, empty, empty, pool.view(2, 4, 2, 32, 64)], **accept)
    with pytest.raises(KernelError, match="given twice"):
        ops.copy_entries([pool, pool.clone(), pool.view(2, 4, -1)], zeros(2), zeros(2), 1)
    assert not ops.names()
    ops.tree_accept(pools=[pool, empty, empty, pool.clone()], **accept)
    ops.copy_entries([pool, empty, empty, pool.clone()], zeros(2), zeros(2), 1)
    assert len(ops.names()) == 2


def test_more_tiles_than_fit_the_row_of_costs_are_refused():
    # 2^12 requests of 2^10 key/value heads, one token, one key: 2^22 blocks of rows; a tile and four more each fit, 511 tiles and as many do not
    R, Hkv = 1 << 12, 1 << 10
    args = dict(q=zeros(1, Hkv, 64, dtype=BF16), k_pool=zeros(1, Hkv, 128, 64, dtype=BF16), v_pool=zeros(1, Hkv, 128, 64, dtype=BF16), cu_q=zeros(R + 1),
                kv_lens=zeros(R), positions=zeros(1), mask=zeros(1, 1), out=zeros(1, Hkv * 64, dtype=BF16), block_table=zeros(R, 507), scale=0.1, window=0,
                page_size=128, max_q_len=1)
    ops = Recorder()
    ops.tree_attention(max_kv_len=1, **args)
    assert ops.names() == ["gb_tree_attention_tc"]
    with pytest.raises(KernelError, match="31 bits"):
        ops.tree_attention(max_kv_len=507 * 128, **args)


def test_pages_without_a_position_and_negative_lengths_are_refused():
    ops = Recorder()
    pool = zeros(4, 2, 0, 64, dtype=BF16)
    with pytest.raises(KernelError, match="at least one position"):
        ops.tree_attention(**attention_args(k_pool=pool, v_pool=pool, page_size=0, max_kv_len=0))
    with pytest.raises(KernelError, match="positions of a request"):
        ops.tree_attention(**attention_args(max_kv_len=-1))
    assert not ops.names()


@pytest.mark.parametrize("hd", [64, 128, 48])
def test_attention_without_heads_or_channels_is_refused(hd):
    """(The kernels divide by the heads of a group.)"""
    ops = Recorder()
    for heads in (0, 2):
        none = zeros(4, heads, 32, hd, dtype=BF16)
        with pytest.raises(KernelError, match="whole groups"):
            ops.tree_attention(**attention_args(q=zeros(5, 0, hd, dtype=BF16), k_pool=none, v_pool=none, out=zeros(5, 0, dtype=BF16)))
    with pytest.raises(KernelError, match="channels"):
        ops.tree_attention(**attention_args(hd=0))
    assert not ops.names()
