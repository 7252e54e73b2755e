"""The argument blocks of the serving calls: the binding's ctypes structures have the
size and the member offsets that a C compiler gives the header's."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("c_name,py_name", [("vvb_kv_plan_t", "KvPlan"), ("vvb_kv_append_slots_t", "KvAppendSlots"),
                                            ("vvb_attn_decode_t", "AttnDecode")])
def test_argument_blocks_agree_with_the_header(tmp_path, c_name, py_name):
    import ctypes

    import vvb200
    st = getattr(vvb200, py_name)
    names = [f[0] for f in st._fields_]
    src = tmp_path / "t.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"vvb200.h\"\nint main(void) {\n"
                   f"  printf(\"%zu\", sizeof({c_name}));\n" +
                   "".join(f"  printf(\" %zu\", offsetof({c_name}, {n}));\n" for n in names) + "  return 0;\n}\n")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(st)] + [getattr(st, n).offset for n in names]
