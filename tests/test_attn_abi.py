"""The attention-side C-ABI (include/lfm_gpu_attn.h) as far as it goes without a GPU."""
import ctypes
import os
import subprocess

import pytest

from laii_b200 import _native, build


def test_exports_every_header_function():
    lib = _native.load_gpu()
    declared = _native.header_functions("lfm_gpu_attn.h", "lfm_gpu_")
    assert len(declared) >= 7
    assert set(declared) == {n for n, _, _ in _native.ATTN_API}
    out = subprocess.run(["nm", "-D", "--defined-only", build.GPU_SO], stdout=subprocess.PIPE, text=True).stdout
    exported = {ln.split()[-1] for ln in out.splitlines() if " T " in ln}
    assert {n for n in exported if n.startswith("lfm_gpu_") and not n.startswith("lfm_gpu_moe_")} == set(declared)
    for name in declared:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("lang", [["gcc", "-std=c11"], ["g++", "-std=c++17"]])
def test_header_compiles(tmp_path, lang):
    src = tmp_path / ("t.c" if lang[0] == "gcc" else "t.cpp")
    src.write_text('#include "lfm_gpu_attn.h"\nint main(void){lfm_gpu_kv_t kv = {0}; lfm_gpu_kv_batch_t b = {0};'
                   ' lfm_gpu_rope_t r = {0}; (void)kv; (void)b; (void)r; return LFM_GPU_OK;}\n')
    r = subprocess.run([*lang, "-Wall", "-Werror", "-I", os.path.join(build.ROOT, "include"), "-c", str(src), "-o",
                        str(tmp_path / "t.o")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout


def test_struct_sizes_match_the_header(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "lfm_gpu_attn.h"\nint main(void){printf("%zu %zu %zu", sizeof(lfm_gpu_kv_t),'
                   ' sizeof(lfm_gpu_kv_batch_t), sizeof(lfm_gpu_rope_t)); return 0;}\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(build.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True).stdout.split()
    assert [int(v) for v in got] == [ctypes.sizeof(t) for t in (_native.Kv, _native.KvBatch, _native.Rope)]


@pytest.mark.parametrize("page,heads,dim,want", [
    (16, 1, 64, 16 * 72), (64, 8, 64, 64 * 8 * 72), (128, 8, 128, 128 * 8 * 144), (32, 1024, 64, 32 * 1024 * 72),
    (0, 8, 64, 0), (8, 8, 64, 0), (48, 8, 64, 0), (256, 8, 64, 0), (64, 0, 64, 0), (64, 1025, 64, 0), (64, 8, 96, 0),
    (64, 8, 0, 0)])
def test_page_bytes(page, heads, dim, want):
    assert _native.load_gpu().lfm_gpu_kv_page_bytes(page, heads, dim) == want


def test_null_handle_is_an_error_not_a_crash():
    lib = _native.load_gpu()
    assert lib.lfm_gpu_add_rmsnorm(None, None, None, 0, 1, 256, None, 1e-5, None, None, 0, None, None) == -1
    assert lib.lfm_gpu_q8k_read(None, None, 1, 256, 0, None, None) == -1
    assert lib.lfm_gpu_kv_append(None, None, None, None, 0, 1, None, 0, None, 0, None, 0, None, 0, None) == -1
    assert lib.lfm_gpu_kv_read(None, None, None, 0, None, None, None) == -1
    assert lib.lfm_gpu_attn_forward(None, None, None, 1, 1.0, 1, 0, 0.0, 0, None, 0, None, 0, None) == -1
    assert lib.lfm_gpu_attn_reserve(None) == -1


def test_python_module_refuses_without_a_launch():
    """Arguments that are not tensors of the device raise before the library is called."""
    import torch
    m = _native.load_attn_py()
    x = torch.zeros(2, 256)
    for x_ in (x, None, 3):
        with pytest.raises(ValueError):
            m.add_rmsnorm(0, 0, x_, None, None, 1e-5, None, -1, True)
    with pytest.raises(ValueError):
        m.read_q8(0, 0, x, 0)
    with pytest.raises(TypeError):
        m.add_rmsnorm(0, 0, None)
    with pytest.raises(TypeError):
        m.read_q8(0, "0", x, 0)
