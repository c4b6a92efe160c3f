"""The cache operators' binding without a GPU: limits, status bits and struct
layouts equal the header's, and calls fail cleanly."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mars_b200.h")


def test_limits_and_bits_match_the_header():
    import mars_b200
    text = open(HEADER).read()
    defines = {m.group(1): int(m.group(2)) for m in re.finditer(r"#define\s+(MARS_[A-Z0-9_]+)\s+(\d+)", text)}
    assert mars_b200.KV_MAX_REQUESTS == defines["MARS_KV_MAX_REQUESTS"]
    bits = {m.group(1): int(m.group(2)) for m in re.finditer(r"\b(MARS_KV_[A-Z_]+)\s*=\s*(\d+)", text)}
    assert len(bits) == 5
    for name, value in bits.items():
        assert getattr(mars_b200, name.replace("MARS_", "")) == value
    types = {m.group(1): int(m.group(2)) for m in re.finditer(r"\bMARS_DTYPE_([A-Z0-9]+)\s*=\s*(\d+)", text)}
    import torch
    from mars_b200 import kv
    assert kv._DTYPES == {torch.float32: types["F32"], torch.float16: types["F16"], torch.bfloat16: types["BF16"]}


def test_struct_layouts_match_the_header(tmp_path):
    from mars_b200 import kv
    structs = {"mars_kv_cache": kv._Cache, "mars_rope_table": kv._Table, "mars_attn_config": kv._Config}
    names = {"mars_kv_cache": None, "mars_rope_table": {"freq": "d_freq", "axis": "d_axis"}, "mars_attn_config": None}
    lines = []
    for c, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        for field, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {(names[c] or {}).get(field, field)}));')
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"mars_b200.h\"\nint main(void) {" + "".join(lines) +
                   "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in structs.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, field).offset for field, _ in py._fields_]
    assert got == want


def test_calls_fail_cleanly_without_a_device():
    import mars_b200
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(mars_b200.MarsError) as e:
        mars_b200.KvContext(max_requests=4)
    assert e.value.status in (mars_b200.MARS_ERR_NO_DEVICE, mars_b200.MARS_ERR_CUDA)
    with pytest.raises(mars_b200.MarsError) as e:
        mars_b200.KvContext(max_requests=0)
    assert e.value.status == mars_b200.MARS_ERR_INVALID
    x = torch.zeros(2, 1, 8)
    with pytest.raises(ValueError):
        mars_b200.rope(x, torch.zeros(2, dtype=torch.int32), torch.ones(4), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        mars_b200.KvCache(torch.zeros(1, 8, 1, 8, dtype=torch.float16), torch.zeros(1, 8, 1, 8, dtype=torch.float16))
