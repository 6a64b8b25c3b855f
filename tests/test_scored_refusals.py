"""Further refusals of the scored attention and the tracked writer, on the host: before any launch."""
import pytest

from rtp_llm_amd import _C
from tests.test_scored_host import _attend, _kv, _write


@pytest.mark.parametrize("kw", [dict(page=1 << 23, hd=128), dict(page=1 << 24, hd=64), dict(page=1 << 24, hd=128, kv_dtype=_C.KV_INT8), dict(page=1 << 25, hd=64, kv_dtype=_C.KV_INT8)])
def test_attention_refuses_heads_of_a_page_beyond_31_bits(kw):
    """A page's keys of one head are addressed by 32-bit offsets in bytes."""
    assert _attend(kv=_kv(num_blocks=1, nkv=4, **kw), ldq=28 * 128) == _C.ERR_ARG
    assert b"page=" in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


@pytest.mark.parametrize("kw", [dict(page=1 << 24, hd=128), dict(page=1 << 25, hd=64), dict(page=1 << 24, hd=128, kv_dtype=_C.KV_INT8)])
def test_writer_refuses_heads_of_a_page_beyond_31_bits(kw):
    """Channels of a page are addressed by 32-bit offsets in elements."""
    assert _write(kv=_kv(num_blocks=1, nkv=4, **kw)) == _C.ERR_ARG
    assert b"page=" in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


@pytest.mark.parametrize("kw", [
    dict(B=32768, rows=32768, nh=8, ldq=1024, kv=_kv(nkv=8), M=1 << 13, most=1 << 17, weights=16),                               # few rows: a thread for four slots of each head
    dict(starts=16, B=4096, rows=4096, q_len=1 << 15, nh=64, ldq=8192, kv=_kv(nkv=8)),                                            # many rows: tiles of the longest sequence for each
    dict(starts=16, B=8192, rows=8192, q_len=64, nh=64, ldq=8192, kv=_kv(nkv=8), M=1 << 13, most=1 << 17, weights=16)])          # ... and blocks of 256 keys
def test_attention_refuses_grids_beyond_32_bits_of_threads(kw):
    assert _attend(**dict(dict(nbytes=1 << 62), **kw)) == _C.ERR_ARG
    assert b"grid" in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()
