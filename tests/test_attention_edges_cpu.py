"""Edges of the cache calls that are settled on the host: no GPU needed."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from test_attention_cpu import _cache
from tritonbench_b200 import lib, ops


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
