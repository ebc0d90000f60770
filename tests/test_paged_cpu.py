"""The paged operators' C entry points refuse bad arguments with a status
before they touch a device, and their ctypes mirrors have the header's sizes."""
import ctypes as C
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_sizes_match_the_header(tmp_path):
    from picchio_b200.paged import _Call, _Pages, _Step
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include "picchio_b200.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   "sizeof(pc_kv_pages), sizeof(pc_kv_step), sizeof(pc_attn_call)); return 0; }\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [C.sizeof(_Pages), C.sizeof(_Step), C.sizeof(_Call)]


def test_bad_arguments_are_refused_without_a_device():
    from picchio_b200.api import lib
    from picchio_b200.paged import _Call, _Pages, _Step, _entry
    lib()
    L = _entry()
    s, p, c = _Step(), _Pages(), _Call()
    two = (C.c_int64 * 2)(64, 64)
    assert L.pc_kv_tables(0, C.byref(s), None) == 1
    assert L.pc_kv_store(0, C.byref(p), 16, two, 16, two, 0, 16, 1, None) == 1
    p.k = p.v = 4096
    p.n_pages, p.n_kv_heads, p.head_dim, p.page_size, p.dtype = 4, 2, 64, 16, 2
    p.ks0 = p.vs0 = 16 * 2 * 64
    p.ks1 = p.vs1 = 2 * 64
    p.ks2 = p.vs2 = 64
    assert L.pc_kv_store(0, C.byref(p), 4096, two, 4096, two, 5, 4096, 1, None) == 3
    assert L.pc_kv_store(0, C.byref(p), 4098, two, 4096, two, 0, 4096, 1, None) == 3
    assert L.pc_kv_store(0, C.byref(p), 4096, two, 4096, two, 0, 4096, 0, None) == 0  # nothing to do
    p.page_size = 12
    assert L.pc_kv_store(0, C.byref(p), 4096, two, 4096, two, 0, 4096, 1, None) == 3
    p.page_size, p.head_dim = 16, 136
    assert L.pc_kv_store(0, C.byref(p), 4096, two, 4096, two, 0, 4096, 1, None) == 3
    assert L.pc_attn_paged(None, C.byref(c), C.byref(p), None, 0, None, None) == 1
    assert L.pc_attn_packed(None, C.byref(c), None, two, None, two, None) == 1
    assert L.pc_attn_create(0, None) == 1
    assert L.pc_attn_check(None, None) == 1
