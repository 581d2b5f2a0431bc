"""The paged 8-bit cache and draft verification without a GPU: refusals that
need no device, and where a token's codes lie (the kernels' own arithmetic,
compiled for the host), bad pages and offsets beyond 32 bits among them."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import hale_pkg

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("kv") / "kv_harness")
    subprocess.run(["g++", "-O1", "-fsanitize=undefined,address", "-static-libasan", "-o", exe,
                    os.path.join(HERE, "kv_harness.cpp")], check=True)

    def ask(**k):
        line = " ".join(str(k[n]) for n in ("n_pages", "nkv", "hd", "log2", "n_seqs", "max_pages", "seq", "pos", "head", "page"))
        out = subprocess.run([exe], input=line, capture_output=True, text=True, check=True).stdout
        return tuple(int(x) for x in out.split())
    return ask


BASE = dict(n_pages=9, nkv=3, hd=48, log2=5, n_seqs=4, max_pages=6, seq=2, pos=70, head=1, page=7)


def test_a_token_lies_where_the_layout_says(harness):
    for pos in (0, 15, 16, 31, 32, 70, 191):
        slot = pos % 32
        assert harness(**{**BASE, "pos": pos}) == (7, ((7 * 3 + 1) * 32 + slot) * 48, ((7 * 3 + 1) * 32 + slot) // 16, slot)


@pytest.mark.parametrize("change", [dict(page=-1), dict(page=9), dict(page=2**31 - 1), dict(page=-2**31), dict(seq=-1),
                                    dict(seq=4), dict(pos=-1), dict(pos=192), dict(pos=2**40)])
def test_a_bad_page_sequence_or_position_names_no_page(harness, change):
    assert harness(**{**BASE, **change})[0] == -1


def test_offsets_pass_32_bits(harness):
    got = harness(n_pages=1 << 20, nkv=8, hd=256, log2=8, n_seqs=1, max_pages=3, seq=0, pos=255, head=7, page=(1 << 20) - 1)
    token = (((1 << 20) - 1) * 8 + 7) * 256 + 255
    assert got == ((1 << 20) - 1, token * 256, token // 16, 255)
    assert token * 256 > 2 ** 38


def test_null_handles_are_refused():
    hale = hale_pkg()
    lib = hale.lib()
    kv = C.byref(hale.Kv8Struct())
    bad = hale.E_INVALID_ARGUMENT
    assert lib.hale_kv8_append(None, kv, 0, None, None, 0, 0, 0, None, None, 1, None) == bad
    assert lib.hale_kv8_read(None, kv, 0, None, None, 1, None, None, 0, 0, 0, None) == bad
    assert lib.hale_kv8_attention(None, kv, 0, None, 0, 0, None, None, 1, 1, 1.0, 0, 1, None, 0, None, None) == bad
    assert lib.hale_kv8_resize(None, kv, None, None, 1, None) == bad
    assert lib.hale_kv8_fork(None, kv, None, None, 1, None) == bad
    assert lib.hale_kv8_compact(None, kv, None, None, None) == bad
    assert lib.hale_kv8_copy(None, kv, None, None, 1, None) == bad
    assert lib.hale_verify_drafts(None, None, 0, 0, None, None, 0, None, 1, 1, 1, 1.0, None, None, None, None, None) == bad
    out = C.c_void_p()
    assert lib.hale_decoder_create_kv8(None, None, None, None, 1, 1, kv, C.byref(out)) == bad
    buf = C.create_string_buffer(128)
    assert lib.hale_last_error(None, buf, 128) == bad and b"NULL" in buf.value
