"""The 8-bit cache's entry points without a GPU: the ctypes structures match the header, and bad arguments are refused before
any device work."""
import ctypes as C
import os
import re
import subprocess
from struct import Struct

import pytest
import torch

import small_llm_b200 as sl
from small_llm_b200 import kv8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
def test_structures_match_the_header(tmp_path):
    lines = []
    for name, (_, fields) in kv8.STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));' for f in fields.split()]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "sllm.h"\nint main(void) {' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), "-o", str(tmp_path / "s")], check=True)
    got = {k: v for k, *v in (line.split() for line in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines())}
    for name, (fmt, fields) in kv8.STRUCTS.items():
        assert int(got[name][0]) == Struct(fmt).size
        at = 0
        for f, letter in zip(fields.split(), "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([A-Za-z])", fmt) if n != "0")):
            size = Struct(letter).size
            at = -(-at // size) * size
            assert [int(x) for x in got[f"{name}.{f}"]] == [at, size], (name, f)
            at += size


def _packed(name, values, over):
    fmt, fields = kv8.STRUCTS[name]
    v = dict(zip(fields.split(), values)) | {k: x or 0 for k, x in over.items()}
    return Struct(fmt).pack(*v.values())


def _layer(**over):
    return _packed("sllm_kv8_layer", (1 << 20, 2 << 20, 4, 2, 64), over)


def _attn(**over):
    return _packed("sllm_kv8_attn", (1 << 24, 1 << 26, 256, 256, 4096, 8192, 8192, 0, 0, 3, 2, 8, 4, 1, 100, 0, 0.0), over)


def _rows(**over):
    return _packed("sllm_kv8_rows", (1 << 24, 1 << 26, 4096, 128, 128, 3, 0), over)


def _refused(fn, *args):
    rc = fn(*args)
    assert rc == 1, rc
    return sl.load_library().sllm_last_error(None).decode()


@pytest.mark.parametrize("over,why", [
    (dict(head_dim=48), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(n_pages=0), "n_pages"),
    (dict(n_pages=1 << 31), "n_pages"), (dict(pages=None), "null"), (dict(scales=None), "null"), (dict(pages=(1 << 20) + 8), "aligned")])
def test_layers_refused(over, why):
    lib = kv8._lib()
    c, got = _layer(**over), C.c_uint64()
    assert why in _refused(lib.sllm_k_kv8_append, c, _rows(), None)
    assert why in _refused(lib.sllm_k_kv8_read, c, _rows(), None)
    assert why in _refused(lib.sllm_k_attn_kv8, c, _attn(), None, 0, None)
    assert why in _refused(lib.sllm_k_attn_kv8_workspace, c, _attn(), C.byref(got))


@pytest.mark.parametrize("over,why", [
    (dict(k=None), "null"), (dict(slot_map=None), "null"), (dict(dtype=2), "dtype"), (dict(k_stride=127), "stride"), (dict(v_stride=1 << 41), "stride"),
    (dict(n_tok=0x40000001), "too many"), (dict(k=(1 << 24) + 1), "misaligned"), (dict(slot_map=4100), "misaligned")])
def test_rows_refused(over, why):
    lib = kv8._lib()
    assert why in _refused(lib.sllm_k_kv8_append, _layer(), _rows(**over), None)
    assert why in _refused(lib.sllm_k_kv8_read, _layer(), _rows(**over), None)


@pytest.mark.parametrize("over,why", [
    (dict(q=None), "null"), (dict(table=None), "null"), (dict(dtype=2), "dtype"), (dict(n_heads=5), "multiple"), (dict(n_heads=0), "multiple"),
    (dict(n_seq=0), "n_seq"), (dict(table_width=0), "table_width"), (dict(q_stride=255), "stride"), (dict(out_stride=255), "stride"),
    (dict(q=(1 << 24) + 1), "misaligned"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(out=(1 << 24) + 512), "overlap"), (dict(tok_pos=8194), "misaligned")])
def test_queries_refused(over, why):
    lib = kv8._lib()
    assert why in _refused(lib.sllm_k_attn_kv8, _layer(), _attn(**over), None, 0, None)


@pytest.mark.parametrize("over,why", [
    (dict(len_before=None), "null"), (dict(slot_map=None), "null"), (dict(n_seq=0), "n_seq"), (dict(n_seq=8193), "n_seq"), (dict(table_width=0), "table_width"),
    (dict(n_pages=0), "n_pages"), (dict(pool_out=4096), "overlap"), (dict(pool_out=4096 + 24), "overlap"), (dict(ring=4098), "misaligned")])
def test_tables_refused(over, why):
    a = _packed("sllm_block_tables", (*[4096] * 5, 8192, *[4096] * 4, 10, 2, 4, 16), over)
    assert why in _refused(kv8._lib().sllm_k_block_tables, a, None)


def test_no_cpu_path():
    with pytest.raises(ValueError, match="no CPU path"):
        kv8.append(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int64), *kv8.empty_cache(1, 1, 64, device="cpu"))
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        kv8.block_tables(z, z, torch.zeros(1, 1, dtype=torch.int32), z, z, z, z, z, z, z)
    with pytest.raises(ValueError, match="head_dim"):
        kv8.empty_cache(1, 1, 80, device="cpu")
    if not torch.cuda.is_available():
        assert kv8._lib().sllm_k_attn_kv8(_layer(), _attn(), None, 0, None) == 3      # SLLM_ERR_CUDA: no device
