"""More of the decoder step's argument blocks: the ctypes mirrors against the header, and the host's checks that need no GPU."""
import ctypes
import os
import subprocess

import pytest

from ingot_amd import KvCache, KvTable, Session
from ingot_amd import _lib as L
from ingot_amd.host import DeviceTensor

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ingot_rocm.h")
STRUCTS = {"ingot_rocm_head_norm": L.HeadNormDesc, "ingot_rocm_kv_prefix": L.KvPrefixDesc,
           "ingot_rocm_verify_args": L.VerifyArgs}


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


def tensor(dtype, *shape):
    return DeviceTensor(None, dtype, shape, 4096, False)


def test_a_call_without_a_session_is_an_error():
    lib = L.load()
    for name, args in (("norm_rotary_apply", [None] * 2 + [0] * 4 + [None] * 2),
                       ("norm_rotary_append", [None] * 6 + [0] * 2 + [None] * 4), ("prefix_attention", [None] * 5),
                       ("verify_drafts", [None])):
        assert getattr(lib, f"ingot_rocm_{name}")(None, *args) == L.EINVAL
        assert "nil session" in lib.ingot_rocm_last_error().decode()


def test_shapes_are_checked_on_the_host():
    """The shapes of every array a kernel reads, before the library is reached."""
    s = Session.__new__(Session)
    s.lib, s.h = L.load(), None
    x, pos, tab = tensor(L.DT_F32, 3, 2, 8), tensor(L.DT_I32, 3), tensor(L.DT_F32, 5, 4)
    for w in (tensor(L.DT_F32, 7), tensor(L.DT_F32, 3, 8), tensor(L.DT_BF16, 8)):
        with pytest.raises(ValueError, match="norm weight"):
            s.prepare_norm_rotary(x, w, pos, tab, tab, x)
    k = tensor(L.DT_BF16, 1, 2, 1, 4, 8)
    cache, table = KvCache(k, k), KvTable(tensor(L.DT_I32, 2, 2), tensor(L.DT_I32, 2))
    kv, starts = tensor(L.DT_F32, 3, 1, 8), tensor(L.DT_I32, 3)
    with pytest.raises(ValueError, match="norm weight"):
        s.prepare_norm_rotary_append(x, kv, kv, None, tensor(L.DT_F32, 2, 8), pos, tab, tab, x, cache, table, starts)
    with pytest.raises(ValueError, match="norm_rotary_append"):
        s.prepare_norm_rotary_append(x, x, kv, None, None, pos, tab, tab, x, cache, table, starts)
    for first, shared in ((tensor(L.DT_I32, 2), tensor(L.DT_I32, 2)), (tensor(L.DT_F32, 2), tensor(L.DT_I32, 1))):
        with pytest.raises(ValueError, match="first"):
            s.prepare_prefix_attention(x, cache, table, starts, x, first, shared)
    with pytest.raises(ValueError, match="prefix_attention mask"):
        s.prepare_prefix_attention(x, cache, table, starts, x, tensor(L.DT_I32, 2), tensor(L.DT_I32, 1),
                                   mask=tensor(L.DT_I32, 4, 1))
    logits, out = tensor(L.DT_F32, 3, 9), (tensor(L.DT_I32, 2, 4), tensor(L.DT_I32, 2), tensor(L.DT_I32, 2))
    good = dict(parents=pos, temperature=tensor(L.DT_F32, 2), accept_u=tensor(L.DT_F32, 3), sample_u=tensor(L.DT_F32, 2))
    s.prepare_verify_drafts(logits, starts, pos, *out, **good)
    for name, bad in (("parents", tensor(L.DT_I32, 2)), ("temperature", tensor(L.DT_F32, 3)),
                      ("accept_u", tensor(L.DT_F32, 2)), ("sample_u", tensor(L.DT_I32, 2)), ("draft", tensor(L.DT_F32, 3, 8))):
        with pytest.raises(ValueError, match=f"verify_drafts {name}"):
            s.prepare_verify_drafts(logits, starts, pos, *out, **{**good, name: bad})
    with pytest.raises(ValueError, match="counts"):
        s.prepare_verify_drafts(logits, starts, pos, out[0], tensor(L.DT_I32, 3), out[2])
