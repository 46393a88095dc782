"""What the rotary, cache-append and cache-attention calls refuse, and the rotary tables: no GPU needed."""
import ctypes
import math

import pytest
import torch

from tritonbench_b200 import lib, ops
from tritonbench_b200.rotary import rotary_frequencies, rotary_table


@pytest.fixture(scope="module")
def cdll():
    return lib.load()


def _cache(p, pages=4, heads=2, size=16, dim=64, pitch=None):
    pitch = pitch or (heads * size * dim, size * dim, dim)
    return lib.KV_CACHE.pack(p, p, p, p, *pitch, *pitch, heads, 1, heads, 1, pages, heads, size, dim)


def _rows(p, width=2, batch=1, tokens=1, cu=0):
    return lib.KV_BATCH.pack(p, p, cu, width, width, batch, tokens)


@pytest.fixture()
def ptr():
    buf = ctypes.create_string_buffer(1 << 12)
    yield (ctypes.addressof(buf) + 255) & ~255  # never dereferenced on the device: every call below is refused before that
    del buf


def test_rotary_refuses_bad_sizes(cdll, ptr):
    def call(x=ptr, dtype=0, y=ptr, tokens=1, heads=1, dim=64, positions=ptr, table=ptr, max_pos=8, rot=64):
        return cdll.b200fp8_rotary(x, dtype, y, tokens, heads, dim, heads * dim, dim, heads * dim, dim, positions, 0, table,
                                   max_pos, rot, 0, 0, None)

    for kw in (dict(x=None), dict(y=None), dict(positions=None), dict(table=None), dict(dtype=3), dict(dtype=-1), dict(rot=63),
               dict(rot=0), dict(rot=66), dict(max_pos=0), dict(heads=0), dict(tokens=-1), dict(dim=0)):
        assert call(**kw) == lib.BAD_ARG, kw
    assert call(tokens=1 << 40) == lib.TOO_LARGE
    assert call(heads=1 << 30) == lib.TOO_LARGE
    assert call(tokens=0) == lib.OK


def test_append_refuses_bad_arguments(cdll, ptr):
    def call(q=ptr, k=ptr, q_out=ptr, dtype=0, heads=4, q_token=256, k_token=128, cache=_cache(ptr), rows=_rows(ptr), table=ptr,
             max_pos=8, rot=64):
        return cdll.b200fp8_kv_append(q, k, k, q_out, dtype, heads, q_token, 64, k_token, 64, k_token, 64, q_token, 64, cache,
                                      rows, table, max_pos, rot, 0, 0, None)

    for kw in (dict(k=None), dict(q_out=None), dict(dtype=2), dict(heads=3), dict(heads=0), dict(cache=None), dict(rows=None),
               dict(rot=0), dict(rot=65), dict(rot=80), dict(max_pos=0), dict(rows=_rows(ptr, tokens=2)),
               dict(rows=_rows(ptr, batch=-1)), dict(rows=_rows(0)), dict(cache=_cache(0)), dict(cache=_cache(ptr, heads=0)),
               dict(rows=_rows(ptr, batch=0, tokens=3, cu=ptr))):
        assert call(**kw) == lib.BAD_ARG, kw
    two = _rows(ptr, batch=2, tokens=2)  # (a pitch that is never used may be odd)
    for kw in (dict(q=ptr + 2), dict(k=ptr + 8), dict(q_token=252, rows=two), dict(k_token=130, rows=two), dict(rot=24), dict(table=ptr + 4),
               dict(cache=_cache(ptr, dim=96)), dict(cache=_cache(ptr, size=24)), dict(cache=_cache(ptr, pitch=(2048, 1024, 72)))):
        assert call(**kw) == lib.UNSUPPORTED_ALIGNMENT, kw
    assert call(rows=_rows(ptr, batch=1 << 30, tokens=1 << 30)) == lib.TOO_LARGE
    assert call(rows=_rows(ptr, width=1 << 28)) == lib.TOO_LARGE
    assert call(rows=_rows(ptr, batch=0, tokens=0)) == lib.OK


def test_attention_refuses_bad_arguments(cdll, ptr):
    def call(q=ptr, out=ptr, dtype=0, heads=4, q_token=256, o_token=256, cache=_cache(ptr), rows=_rows(ptr), ws=ptr):
        return cdll.b200fp8_kv_attention(q, out, None, dtype, heads, q_token, 64, o_token, 64, cache, rows, 0.125, 0, ws, 16, None)

    for kw in (dict(q=None), dict(out=None), dict(dtype=2), dict(heads=5), dict(cache=None), dict(rows=None),
               dict(rows=_rows(ptr, tokens=2)), dict(rows=_rows(0))):
        assert call(**kw) == lib.BAD_ARG, kw
    two = _rows(ptr, batch=2, tokens=2)
    for kw in (dict(q=ptr + 8), dict(out=ptr + 4), dict(q_token=260, rows=two), dict(o_token=258, rows=two), dict(ws=ptr + 8),
               dict(cache=_cache(ptr, dim=32)), dict(cache=_cache(ptr, size=256))):
        assert call(**kw) == lib.UNSUPPORTED_ALIGNMENT, kw
    assert call(rows=_rows(ptr, batch=0, tokens=0)) == lib.OK
    assert cdll.b200fp8_kv_attention_workspace_bytes(None, _rows(ptr), 4) == 0
    assert cdll.b200fp8_kv_attention_workspace_bytes(_cache(ptr, dim=96), _rows(ptr), 4) == 0


def test_the_wrappers_take_no_cpu_tensors():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary(x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.Fp8KvCache.empty(2, 2, 64, device="cpu")
    for call in (lambda: ops.fp8_kv_append(x, x, x, None, None, None), lambda: ops.fp8_kv_attention(x, None, None, None)):
        with pytest.raises(ValueError, match="Fp8KvCache"):
            call()


# ------------------------------------------------------------------ tables
def test_table_holds_cosines_and_sines_of_64_bit_angles():
    table = rotary_table(100_003, 64, base=500.0)
    pos = torch.tensor([0, 1, 7, 65_537, 100_002])
    want = pos.double()[:, None] * torch.tensor([500.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    # half a step of fp32 at one, and two 64-bit roundings of an angle below 1e5 (2 * 1e5 * 2^-53)
    assert (table[pos, :32].double() - want.cos()).abs().max() < 2**-25 + 1e-10
    assert (table[pos, 32:].double() - want.sin()).abs().max() < 2**-25 + 1e-10


def test_scaled_frequencies_keep_fast_pairs_and_stretch_slow_ones():
    plain, gain = rotary_frequencies(128)
    assert gain == 1.0 and plain[0] == 1.0
    linear, _ = rotary_frequencies(128, scaling="linear", factor=4.0)
    assert torch.equal(linear, plain / 4)
    ntk, _ = rotary_frequencies(128, scaling="ntk", factor=4.0)
    assert ntk[0] == plain[0] and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    yarn, gain = rotary_frequencies(128, scaling="yarn", factor=4.0, original_max=4096)
    assert math.isclose(gain, 0.1 * math.log(4.0) + 1)
    assert torch.equal(yarn[:16], plain[:16]) and torch.equal(yarn[-10:], plain[-10:] / 4)
    assert ((yarn <= plain) & (yarn >= plain / 4)).all()
    banded, gain = rotary_frequencies(128, scaling="banded", factor=8.0, original_max=8192)
    turns = 8192 * plain / (2 * math.pi)
    assert gain == 1.0
    assert torch.equal(banded[turns > 4], plain[turns > 4]) and torch.equal(banded[turns < 1], plain[turns < 1] / 8)
    for i in torch.nonzero((turns > 1) & (turns < 4)).flatten().tolist():
        keep = (float(turns[i]) - 1) / 3
        assert math.isclose(banded[i], plain[i] * keep + plain[i] / 8 * (1 - keep), rel_tol=1e-12)


def test_table_gain_multiplies_both_parts():
    table = rotary_table(8, 32, scaling="yarn", factor=16.0)
    gain = 0.1 * math.log(16.0) + 1
    assert (table[0, :16].double() - gain).abs().max() < gain * 2**-24 + 1e-15
    assert table[0, 16:].abs().max() == 0


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=64, factor=0.0), dict(rot_dim=64, scaling="other"),
                                dict(rot_dim=64, base=0.0), dict(rot_dim=2, scaling="ntk", factor=2.0),
                                dict(rot_dim=64, scaling="banded", low=4.0, high=1.0), dict(rot_dim=64, scaling="yarn", original_max=0)])
def test_table_refuses(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)
