"""Edges of the cache calls that are settled on the host: no GPU needed."""
import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from test_attention_cpu import _cache
from tritonbench_b200 import lib, ops
from tritonbench_b200.rotary import rotary_frequencies


@pytest.fixture(scope="module")
def cdll():
    return lib.load()


@pytest.fixture()
def ptr():
    buf = ctypes.create_string_buffer(1 << 12)
    yield (ctypes.addressof(buf) + 255) & ~255  # never dereferenced on the device: every call below is refused before that
    del buf


@pytest.mark.parametrize("rows,pitch", [(torch.arange(7, dtype=torch.int32).expand(3, 7), 0),
                                        (torch.arange(20, dtype=torch.int32).as_strided((3, 7), (2, 1)), 2),
                                        (torch.arange(30, dtype=torch.int32).view(3, 10)[:, :7], 10)])
def test_rows_of_the_block_table_lie_where_its_stride_says(rows, pitch):
    """Rows that overlap or are one: the device must not be told that they lie a row's width apart."""
    packed = ops._pack_batch(3, SimpleNamespace(device=-1), rows, torch.ones(3, dtype=torch.int32), None)
    table, _, _, table_pitch, width, batch, tokens = lib.KV_BATCH.unpack(packed)
    assert (table, table_pitch, width, batch, tokens) == (rows.data_ptr(), pitch, 7, 3, 3)


def test_table_pitches_that_the_library_takes(cdll, ptr):
    def call(pitch, width=2):
        rows = lib.KV_BATCH.pack(ptr, ptr, 0, pitch, width, 2, 2)
        cache = _cache(ptr, pitch=(2048, 1024, 72))  # refused, but after the batch
        return cdll.b200fp8_kv_attention(ptr, ptr, None, 0, 4, 256, 64, 256, 64, cache, rows, 0.125, 0, ptr, 16, None)

    assert call(-1) == lib.BAD_ARG
    assert call(0) == call(1) == call(2) == lib.UNSUPPORTED_ALIGNMENT
    assert call(1 << 40, width=1 << 60) == lib.TOO_LARGE


def test_append_refuses_pitches_of_zero(cdll, ptr):
    """One scale, or one row of codes, of several pages or heads would be read and written by several blocks at once."""
    def call(pitches, scale_pitches, pages=4, heads=2):
        cache = lib.KV_CACHE.pack(ptr, ptr, ptr, ptr, *pitches, *pitches, *scale_pitches, *scale_pitches, pages, heads, 16, 64)
        rows = lib.KV_BATCH.pack(ptr, ptr, 0, 2, 2, 1, 1)
        # q on an odd address: refused, but after the cache
        return cdll.b200fp8_kv_append(ptr + 2, ptr, ptr, ptr, 0, 4, 256, 64, 128, 64, 128, 64, 256, 64, cache, rows, None, 0, 0, 0, 0, None)

    good, scales = (2048, 1024, 64), (2, 1)
    assert call(good, scales) == lib.UNSUPPORTED_ALIGNMENT
    for i in range(3):
        assert call([0 if i == j else p for j, p in enumerate(good)], scales) == lib.BAD_ARG
    assert call(good, (0, 1)) == call(good, (2, 0)) == lib.BAD_ARG
    assert call((0, 0, 64), (0, 0), pages=1, heads=1) == lib.UNSUPPORTED_ALIGNMENT  # pitches that are never used


def test_tensors_whose_elements_are_one():
    x = torch.zeros(4, 3, 16, 64)
    for t in (x, x.transpose(1, 2), x[:, 1:2], x[::2, :, :, ::4], x[..., :48], x.unflatten(0, (2, 2))[:, 1], torch.zeros(1).expand(1, 1)):
        assert not ops._elements_share_memory(t)
    for t in (x[:1].expand(4, 3, 16, 64), x[:, :1].expand(4, 3, 16, 64), torch.zeros(4, 1).expand(4, 3), torch.zeros(1).expand(2),
              torch.zeros(200).as_strided((3, 64), (32, 1))):
        assert ops._elements_share_memory(t)


@pytest.mark.parametrize("base", [1.0, 0.5])
def test_yarn_refuses_bases_whose_pairs_do_not_slow_down(base):
    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(8, base=base, scaling="yarn", factor=4.0)
    assert rotary_frequencies(8, base=base, scaling="linear", factor=4.0)[0].isfinite().all()


@pytest.mark.parametrize("original_max", [1, 5, 6, 7, 100, 300, 10**12])
@pytest.mark.parametrize("rot", [2, 8, 128])
def test_yarn_stretches_what_turns_less_than_once(rot, original_max):
    plain, _ = rotary_frequencies(rot)
    freq, _ = rotary_frequencies(rot, scaling="yarn", factor=4.0, original_max=original_max)
    turns = original_max * plain / (2 * math.pi)
    # the ramp begins and ends on whole pairs: one pair beyond either limit may lie on it
    slow, fast = turns < 10000.0 ** (-2 / rot), turns > 32 * 10000.0 ** (2 / rot)
    if original_max < 6:
        slow = turns < 1
    assert torch.equal(freq[slow], plain[slow] / 4) and torch.equal(freq[fast], plain[fast])
    assert ((freq <= plain) & (freq >= plain / 4)).all()
