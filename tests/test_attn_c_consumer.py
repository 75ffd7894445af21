"""include/sera_attn.h from a C99 caller: compiles alone with -std=c99 -Wall -Wextra -Werror -pedantic, has the layout that
the Python structures assume, and its host-side answers are those of the Python calls. No GPU is touched."""
import ctypes
import os
import shutil
import subprocess

import pytest

import q3q4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "sera_attn.h"
#include "sera_q4k.h"
#include <stdio.h>

int main(void) {
    static int32_t row_start[3] = {0, 512, 513}, kv_len[2] = {512, 700}, page_table[22];
    static unsigned char data[16];
    sera_kv_cache cache = {SERA_KV_Q8, /* tokens a page */ 64, /* kv heads */ 8, /* channels */ 128, 4, data};
    sera_kv_batch batch = {2, 513, 512, 700, 11, row_start, kv_len, page_table};
    printf("sizes %zu %zu %zu %zu\n", sizeof cache, offsetof(sera_kv_cache, data), sizeof batch,
           offsetof(sera_kv_batch, row_start));
    printf("page %zu %zu\n", sera_kv_page_bytes(SERA_KV_Q8, 64, 8, 128), sera_kv_page_bytes(SERA_KV_F16, 48, 8, 128));
    printf("workspace %zu\n", sera_attention_workspace_bytes(&cache, &batch, 64));
    printf("write %d\n", sera_kv_write(&cache, &batch, SERA_TYPE_F32, 0, 1024, 0, 1024, 0));
    printf("error %s\n", sera_q4k_last_error());
    printf("read %d\n", sera_kv_read(&cache, &batch, 7u, data, 1024, data, 1024, 0));
    printf("attention %d\n", sera_attention(&cache, &batch, SERA_TYPE_BF16, data, 8192, data, 8192, 60, 0.1f, 0, 0, 0, 0, 0));
    return 0;
}
"""


def cc():
    found = shutil.which("gcc") or shutil.which("cc")
    if found is None:
        pytest.fail("no C compiler in PATH")
    return [found, "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include")]


def test_header_compiles_alone(tmp_path):
    src = tmp_path / "alone.c"
    src.write_text('#include "sera_attn.h"\n#include "sera_attn.h"\nint unused;\n')
    r = subprocess.run(cc() + ["-c", str(src), "-o", str(tmp_path / "alone.o")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


def test_c99_caller_compiles_links_and_runs(tmp_path):
    L = q3q4.load()
    src, exe = tmp_path / "caller.c", tmp_path / "caller"
    src.write_text(SOURCE)
    libdir = os.path.dirname(q3q4.LIB_PATH)
    r = subprocess.run(cc() + [str(src), "-L", libdir, "-lsera_q4k", f"-Wl,-rpath,{libdir}", "-o", str(exe)],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = dict(line.split(" ", 1) for line in r.stdout.strip().splitlines())
    C, B = q3q4.KVCacheArgs, q3q4.KVBatchArgs
    assert out["sizes"] == f"{ctypes.sizeof(C)} {C.data.offset} {ctypes.sizeof(B)} {B.row_start.offset}"
    assert out["page"] == f"{8 * (64 * 128 * 2 + 64 * 8)} 0"
    c, b = C(q3q4.KV_Q8, 64, 8, 128, 4, 16), B(2, 513, 512, 700, 11, 4, 4, 4)
    assert out["workspace"] == str(L.sera_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 64))
    assert out["write"] == out["read"] == out["attention"] == "-1"
    assert "sera_kv_write" in out["error"] and "null k" in out["error"]
