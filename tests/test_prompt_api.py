"""CPU-side checks of the prompt and shared-prefix calls: the ctypes structs
have the C layout, a null context is refused before any CUDA call, and the
binding refuses host tensors."""
import ctypes as C
import os
import shutil
import subprocess
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_is_the_headers(tmp_path):
    import k3xb
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    structs = {"k3xb_kv_rows": k3xb.KvRows, "k3xb_prefix_attention_io": k3xb.PrefixAttentionIO}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "k3xb.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in structs.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
    assert k3xb._IO.size == C.sizeof(k3xb.PrefixAttentionIO)


def test_null_context_is_refused():
    import k3xb
    lib = k3xb.library()
    assert lib.k3xb_kda_prefill(None, *[None] * 3, 0, 0, None, None, None, 1, 1, 1, 128, None, None, None) == k3xb.INVALID_EXTENT
    assert lib.k3xb_kda_step(None, *[None] * 3, 0, 0, None, None, 1, 1, 128, None, 1, None, None) == k3xb.INVALID_EXTENT
    assert lib.k3xb_prefix_attention(None, C.byref(k3xb.PrefixAttentionIO())) == k3xb.INVALID_EXTENT


def test_host_tensors_are_refused():
    import torch

    import k3xb
    q = torch.zeros(2, 64)
    with pytest.raises(k3xb.K3xbError) as e:
        k3xb.Context._kda_rows(types.SimpleNamespace(device=0), q, q, q, q, torch.zeros(2, 1), q)
    assert e.value.status == k3xb.INVALID_EXTENT
    k = torch.zeros(1, 4, 2, 64)
    with pytest.raises(k3xb.K3xbError) as e:
        k3xb.Context._kv_rows(k, k, None, (1,), 2, 64, 64, 0, torch.float32, 0)
    assert e.value.status == k3xb.INVALID_EXTENT


@pytest.mark.parametrize("q,k,v", [((2, 4, 64), (2, 9, 4, 64), (2, 9, 4, 64)), ((2, 1, 4, 64), (2, 9, 64), (2, 9, 4, 64)),
                                   ((2, 1, 4, 64), (2, 9, 4, 64), (9, 4, 64))])
def test_other_ranks_are_refused(q, k, v):
    import torch

    import k3xb
    ctx = types.SimpleNamespace(device=0)
    with pytest.raises(k3xb.K3xbError) as e:
        k3xb.Context.prefix_attention(ctx, torch.zeros(q), None, None, torch.zeros(k), torch.zeros(v), None, [-1], None)
    assert e.value.status == k3xb.INVALID_EXTENT


@pytest.mark.parametrize("v", [None, (9, 4)])
def test_a_prefix_without_values_is_refused(v):
    import torch

    import k3xb
    with pytest.raises(k3xb.K3xbError) as e:
        k3xb.Context._kv_rows(torch.zeros(9, 4, 64), v and torch.zeros(v), None, (), 4, 64, 64, 0, torch.float32, 0)
    assert e.value.status == k3xb.INVALID_EXTENT
