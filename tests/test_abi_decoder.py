"""The decoder step's argument blocks: the ctypes mirrors against the header, and the host's checks that need no GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from ingot_amd import Heads, KvCache, KvTable
from ingot_amd import _lib as L
from ingot_amd.host import DeviceTensor

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ingot_rocm.h")
STRUCTS = {"ingot_rocm_kv_cache": L.KvCacheDesc, "ingot_rocm_kv_table": L.KvTableDesc, "ingot_rocm_kv_batch": L.KvBatchDesc,
           "ingot_rocm_heads": L.HeadsDesc, "ingot_rocm_rotary": L.RotaryDesc,
           "ingot_rocm_rotary_table_args": L.RotaryTableArgs, "ingot_rocm_tree_attention_args": L.TreeAttentionArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void){{\n' + "\n".join(lines)
                   + "\nreturn 0;}\n")
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    out = iter(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    for name, mirror in STRUCTS.items():
        assert ctypes.sizeof(mirror) == int(next(out)), name
        for f in mirror._fields_:
            assert getattr(mirror, f[0]).offset == int(next(out)), f"{name}.{f[0]}"


def tensor(dtype, shape):
    return DeviceTensor(None, dtype, shape, 4096, False)


def test_views_of_heads():
    t = tensor(L.DT_BF16, (3, 100))
    h = Heads(t, 3, 2, 8, 20, 100, 8)
    assert (h.c.data, h.c.token, h.c.head) == (4096 + 40, 100, 8)
    for args in ((3, 2, 8, 85, 100, 8), (3, 2, 8, -1, 100, 8), (4, 2, 8, 20, 100, 8), (3, 2, 8, 20, -100, 8)):
        with pytest.raises(ValueError, match="view"):
            Heads(t, *args)
    with pytest.raises(ValueError, match="tokens, heads, dim"):
        Heads(t)
    assert Heads(tensor(L.DT_F32, (0, 2, 8))).tokens == 0


def test_caches_and_tables():
    k = tensor(L.DT_BF16, (2, 5, 3, 16, 8))
    a, b = KvCache(k, k).c, KvCache(tensor(L.DT_BF16, (2, 5, 16, 3, 8)), tensor(L.DT_BF16, (2, 5, 16, 3, 8)), True).c
    for c in (a, b):
        assert (c.kv_heads, c.head_dim, c.page_size, c.layers, c.pages) == (3, 8, 16, 2, 5)
        assert (c.stride_layer, c.stride_page) == (5 * 384, 384)
    assert (a.stride_head, a.stride_slot) == (128, 8) and (b.stride_head, b.stride_slot) == (8, 24)
    with pytest.raises(ValueError, match="alike"):
        KvCache(k, tensor(L.DT_F32, k.shape))
    pages, lengths = tensor(L.DT_I32, (4, 6)), tensor(L.DT_I32, (4,))
    assert (KvTable(pages, lengths).c.rows, KvTable(pages, lengths).c.max_pages) == (4, 6)
    with pytest.raises(ValueError, match="table"):
        KvTable(pages, tensor(L.DT_I32, (5,)))
    with pytest.raises(ValueError, match="int32"):
        KvTable(pages, tensor(L.DT_I64, (4,)))


def test_example_drafts():
    """The example's host side: trees that list parents first, and the path the logits take through one."""
    import importlib.util
    path = os.path.join(os.path.dirname(HEADER), "..", "examples", "speculative_decoding.py")
    spec = importlib.util.spec_from_file_location("speculative_decoding", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    tree = ex.draft_tree([1, 2, 3, 1, 4, 1, 2, 1], depth=3, breadth=2, nodes=6)
    assert tree[:3] == [(1, -1, 0), (2, 0, 1), (4, 0, 1)] and len(tree) == 6
    assert all(parent < i for i, (_, parent, _) in enumerate(tree))
    logits = np.zeros((6, 9))
    logits[0, 4] = logits[2, 1] = 1.0
    child = next(i for i, n in enumerate(tree) if n[:2] == (1, 2))
    logits[child, 8] = 1.0
    assert ex.longest_path(tree, logits) == ([0, 2, child], 8)
