"""A library built from older sources, given by its path: it loads, the operators that it has run, those that it lacks raise and name
what is missing, and the routing does without them. The stand-in here exports names alone and none of them is called.
"""
import shutil
import subprocess

import pytest
import torch

from mi50_vllm_lab_amd import pth_dec
from mi50_vllm_lab_amd import vllm_shim as shim


@pytest.fixture
def older(tmp_path, monkeypatch):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")

    def make(missing):
        src, lib = tmp_path / f"stub{len(missing)}.c", tmp_path / f"libstub{len(missing)}.so"
        src.write_text("\n".join(f"int {n}(void) {{ return 0; }}" for n in pth_dec.EXPORTED_SYMBOLS if n not in missing))
        subprocess.run([cc, "-shared", "-fPIC", str(src), "-o", str(lib)], check=True)
        monkeypatch.setenv("VLLM_GFX950_PTH_DEC_LIB", str(lib))
        monkeypatch.setenv("VLLM_GFX950_PTH_FA_LIB", str(lib))
        shim.reset_loaders()
        return str(lib)

    yield make
    shim.reset_loaders()
    pth_dec.load_library(pth_dec.LIB_PATH)
    assert all(map(pth_dec.provides, pth_dec.LATER_SYMBOLS))


def layer(**kw):
    return shim.Gfx950Int8Attention(**{**dict(num_heads=24, num_kv_heads=4, head_size=256, scale=1 / 16, kv_quant_int8_per_token_head=True,
                                              is_rocm=True, is_decoder=True, sliding_window=(1023, -1)), **kw})


def test_it_loads_and_what_it_lacks_raises(older):
    lib = pth_dec.load_library(older(pth_dec.LATER_SYMBOLS))
    assert pth_dec.provides("pth_dec_decode") and pth_dec.provides("pth_cache_evict")
    assert not any(map(pth_dec.provides, pth_dec.LATER_SYMBOLS)) and lib.pth_dec_decode.argtypes
    x = torch.zeros((3, 8, 256), dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="has no pth_fa_forward_window"):
        pth_dec.forward_window(x, x, x, i, i, 1.0, i, x, 16)
    with pytest.raises(RuntimeError, match="has no pth_cache_fork_pages"):
        pth_dec.fork_pages([x], i, i, i, None, i, i, i, i)
    with pytest.raises(RuntimeError, match="has no pth_cache_compact_pages"):
        pth_dec.compact_pages([x], i, i, i, i, i, i)
    with pytest.raises(RuntimeError, match="has no pth_cache_write_norm_rotary"):
        pth_dec.norm_rotary_cache_write(x, x, x, x, x, i, x, x, x, x, x, i)


def test_windowed_layers_keep_decode_and_leave_prefill(older):
    older(pth_dec.LATER_SYMBOLS)
    a = layer()
    assert a.pth_dec is not None and a.pth_fa_window is None
    assert layer(sliding_window=(-1, -1)).pth_fa is not None
    with pytest.raises(RuntimeError, match="sink_tokens"):
        layer(sink_tokens=4)


def test_decode_without_sinks_leaves_their_rows_to_forward_window(older):
    older(("pth_dec_decode_sinks",))
    a = layer(sink_tokens=4)
    assert a.pth_dec is None and a.pth_fa_window is not None and layer().pth_dec is not None


def test_a_library_without_the_first_entries_is_none(older):
    with pytest.raises(AttributeError):
        pth_dec.load_library(older(("pth_dec_decode",)))
    assert layer().pth_dec is None


def test_addresses_are_the_active_library_s(older):
    """not those that an earlier one left."""
    pth_dec.load_library()
    before = pth_dec._entry("pth_fa_forward_window")
    older_path = older(("pth_fa_forward_window",))
    pth_dec.load_library(older_path)
    assert not pth_dec.provides("pth_fa_forward_window")
    pth_dec.load_library(pth_dec.LIB_PATH)
    assert pth_dec._entry("pth_fa_forward_window") == before
