"""The cache's structures as calls send them, as ctypes declares them and as include/hmx.h does:
one layout (CPU)."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from hmx import _lib

INCLUDE = Path(__file__).resolve().parent.parent / "include"


@pytest.mark.parametrize("layout,name", [(_lib.PagedKV, "hmx_paged_kv"), (_lib.KVScales, "hmx_kv_scales")])
def test_fields_lie_where_the_header_has_them(tmp_path, layout, name):
    fields = [f for f, _ in layout._fields_]
    src = "#include <stddef.h>\n#include <stdint.h>\n#include \"hmx.h\"\nint64_t at[] = {%s, sizeof(%s)};\n" % (
        ", ".join(f"offsetof({name}, {f})" for f in fields), name)
    (tmp_path / "at.c").write_text(src)
    subprocess.run(["gcc", "-shared", "-fPIC", f"-I{INCLUDE}", "-o", str(tmp_path / "at.so"), str(tmp_path / "at.c")], check=True)
    at = (ctypes.c_int64 * (len(fields) + 1)).in_dll(ctypes.CDLL(str(tmp_path / "at.so")), "at")
    assert list(at) == [getattr(layout, f).offset for f in fields] + [ctypes.sizeof(layout)]


def test_what_calls_send():
    k, v = (torch.zeros(5, 3, 16, 64, dtype=torch.uint8).transpose(1, 2) for _ in range(2))
    table, lens = torch.zeros(4, 9, dtype=torch.int32)[:, :7], torch.zeros(4, dtype=torch.int32)
    got = _lib.PagedKV.from_buffer_copy(_lib.paged_kv(k, v, table, lens))
    want = dict(k=k.data_ptr(), k_page_stride=3 * 16 * 64, k_token_stride=64, k_head_stride=16 * 64,
                v=v.data_ptr(), v_page_stride=3 * 16 * 64, v_token_stride=64, v_head_stride=16 * 64,
                table=table.data_ptr(), table_stride=9, seq_lens=lens.data_ptr(), table_width=7, num_pages=5, page_size=16)
    assert {f: getattr(got, f) for f, _ in got._fields_} == want
    bare = _lib.PagedKV.from_buffer_copy(_lib.paged_kv(k, v))
    assert (bare.table, bare.table_stride, bare.seq_lens, bare.table_width, bare.page_size) == (None, 0, None, 0, 16)
    ks, vs = torch.zeros(5, 3, 16, dtype=torch.uint8), torch.zeros(5, 4, 20, dtype=torch.uint8)[:, 1:, :16]
    got = _lib.KVScales.from_buffer_copy(_lib.kv_scales(ks, vs))
    want = dict(k=ks.data_ptr(), k_page_stride=48, k_head_stride=16, v=vs.data_ptr(), v_page_stride=80, v_head_stride=20)
    assert {f: getattr(got, f) for f, _ in got._fields_} == want
