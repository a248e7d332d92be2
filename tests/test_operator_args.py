"""The norm + append, shared-prefix and 4-bit entry points refuse bad arguments
before any CUDA call (the addresses below are never touched)."""
import ctypes as C
import os

import pytest

from hxinfer_b200 import _lib

BAD, OK = _lib.HX_ERR_INVALID, _lib.HX_OK
FP16, FP32, BF16 = _lib.HX_FP16, _lib.HX_FP32, _lib.HX_BF16
A, B, D, E = 0x10000, 0x20000, 0x30000, 0x40000


@pytest.mark.parametrize("out,inp,group", [(0, 128, 128), (16, 0, 128), (16, 128, 16), (16, 96, 64),
                                           (16, 160, 128), (16, 128, 0), (16, 128, -32),
                                           (-1, 128, 32), (16, 100, 32), (16, 256, 256)])
def test_w4_sizes(hxlib, out, inp, group):
    assert hxlib.hx_w4_packed_bytes(out, inp, group, 0) == 0
    assert hxlib.hx_w4_pack(A, B, None, out, inp, group, D, 1 << 30, None) == BAD
    assert hxlib.hx_w4_quantize(A, out, inp, group, B, D, None) == BAD
    assert hxlib.hx_w4_linear(A, 1, inp, B, 1 << 30, out, group, 0, None, D, FP16, None) == BAD


@pytest.mark.parametrize("out,inp,group,zeros,want", [
    (16, 128, 128, 0, 1024 + 32),            # one tile, one unit
    (17, 128, 128, 0, 2 * (1024 + 32)),      # rows in tiles of 16
    (16, 160, 32, 0, 2048 + 8 * 32),         # inputs in units of 128
    (16, 128, 32, 1, 1024 + 4 * (32 + 16)),
    (1 << 17, 1 << 16, 128, 0, (1 << 32) + (1 << 27)),   # past 32 bits
])
def test_w4_packed_bytes(hxlib, out, inp, group, zeros, want):
    assert hxlib.hx_w4_packed_bytes(out, inp, group, zeros) == want


def test_w4_pointers_and_dtypes(hxlib):
    need = hxlib.hx_w4_packed_bytes(16, 128, 128, 0)
    lin = hxlib.hx_w4_linear
    assert lin(A, 0, 128, B, need, 16, 128, 0, None, D, FP16, None) == OK     # nothing to do
    assert lin(A, -1, 128, B, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 65535 * 32 + 1, 128, B, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need - 1, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 1, None, D, FP16, None) == BAD    # zero points need more
    assert lin(A + 8, 1, 128, B, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B + 8, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 0, E + 1, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 0, None, D + 2, FP32, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 0, None, D, BF16, None) == BAD
    assert lin(None, 1, 128, B, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 0, None, A, FP16, None) == BAD    # y over x
    assert lin(A, 3, 128, B, need, 16, 128, 0, None, A + 3 * 256 - 2, FP16, None) == BAD
    assert lin(D + 32, 1, 128, B, need, 16, 128, 0, None, D, FP32, None) == BAD
    assert lin(A, 1, 128, None, need, 16, 128, 0, None, D, FP16, None) == BAD
    assert lin(A, 1, 128, B, need, 16, 128, 0, None, None, FP16, None) == BAD
    pack = hxlib.hx_w4_pack
    assert pack(A, B, None, 16, 128, 128, D, need - 1, None) == BAD
    assert pack(A, B, None, 16, 128, 128, D + 8, need, None) == BAD
    assert pack(A, B + 1, None, 16, 128, 128, D, need, None) == BAD
    assert pack(None, B, None, 16, 128, 128, D, need, None) == BAD
    assert pack(A, None, None, 16, 128, 128, D, need, None) == BAD
    assert hxlib.hx_w4_quantize(A, 16, 128, 128, None, D, None) == BAD
    assert hxlib.hx_w4_quantize(A + 1, 16, 128, 128, B, D, None) == BAD


def test_packed_spec_has_the_header_s_layout(tmp_path):
    """The fields' offsets and the size of hx_norm_append_spec, by the C compiler."""
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not present")
    names = ["q", "k", "v", "q_stride", "k_stride", "v_stride", "q_weight", "k_weight", "seq_ids", "positions",
             "table", "q_out", "dtype", "q_out_dtype", "n_tokens", "num_q_heads", "eps"]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "hx_kv.h"\nint main(void) {\n' +
                   "".join(f'    printf("%zu ", offsetof(hx_norm_append_spec, {n}));\n' for n in names) +
                   '    printf("%zu", sizeof(hx_norm_append_spec));\n    return 0;\n}\n')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "layout"
    subprocess.run([gcc, f"-I{os.path.join(root, 'include')}", str(src), "-o", str(exe)], check=True)
    offsets = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    want, at = [], 0
    for code in "PPPqqqPPPPPPiiiif":
        want.append(at)
        at += 4 if code in "if" else 8
    assert offsets == want + [_lib.norm_append_spec.size]


def test_null_caches_and_tables(hxlib):
    out = C.c_void_p()
    spec = _lib.norm_append_spec.pack(A, A, A, 128, 128, 128, 0, 0, B, B, 0, D, FP16, FP16, 1, 1, 1e-6)
    assert hxlib.hx_norm_rope_append(None, 0, spec, None) == BAD
    assert hxlib.hx_decode_attention_shared(None, 0, A, B, B, 1, 1, 0, 0, 1.0, D, FP16, E, 64,
                                            None) == BAD
    assert hxlib.hx_decode_shared_workspace_bytes(None, 1, 1, 0) == 0
    assert hxlib.hx_kv_share(None, 0, 1, 0, None) == BAD
    make = hxlib.hx_rope_table_create_values
    for hd, n, c, s in ((128, 4, None, B), (128, 4, A, None), (127, 4, A, B), (0, 4, A, B),
                        (258, 4, A, B), (128, 0, A, B)):
        assert make(hd, n, c, s, None, C.byref(out)) == BAD
        assert not out.value
    assert make(128, 4, A, B, None, None) == BAD
