"""Paged 8-bit KV cache without a GPU: what the C entry points refuse, and the
oracle's own properties."""
import ctypes as C
import math

import numpy as np
import pytest

from lowbit_b200 import kernels as K
from lowbit_b200.kvcache import _KV8
from oracle import kv8_ref as R

A = 1 << 20  # an aligned address; refused calls touch no memory


def pool(**over):
    f = dict(k=A, v=A, k_exp=A, v_exp=A, page_stride=2 * 64 * 64, exp_stride=2, pages=4, page=64, kv_heads=2, head_dim=64)
    f.update(over)
    return C.byref(_KV8(*(f[n] for n, _ in _KV8._fields_)))


@pytest.mark.parametrize("over", [
    dict(k=None), dict(v_exp=None), dict(page=48), dict(page=0), dict(head_dim=96), dict(pages=0), dict(kv_heads=0),
    dict(page_stride=2 * 64 * 64 - 16), dict(page_stride=2 * 64 * 64 + 8), dict(exp_stride=1), dict(k=A + 8)])
def test_c_entries_refuse_bad_pools(over):
    L = K.lib()
    for rc in (L.lbc_kv8_read(pool(**over), 1, A, 1, A, A, None),
               L.lbc_kv8_attention(pool(**over), 0, A, 256, A, 4, A, None, 1, 1, 1, 4, 0, 0.125, A, None, 0, None),
               L.lbc_kv8_append(pool(**over), 0, A, 512, None, A, A, 64, A, 4, A, None, 1, 1, 1, 4, A, None)):
        assert rc == -1
        assert b"kv8" in L.lbc_last_error()


def test_c_entries_refuse_null_pools():
    L = K.lib()
    assert L.lbc_kv8_read(None, 1, A, 1, A, A, None) == -1
    assert L.lbc_kv8_attention_workspace(None, 0, 4, 1, 1, 1, 4, 0) == 0


def test_python_refuses_host_tensors():
    import torch

    import lowbit_b200 as lb
    k = torch.zeros((4, 2, 64, 64), dtype=torch.int8)
    e = torch.zeros((4, 2), dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        lb.KV8Cache(k, k.clone(), e, e.clone())
    with pytest.raises(ValueError, match="int8"):
        lb.KV8Cache(k.float(), k.float(), e, e)
    with pytest.raises(ValueError, match="uint8"):
        lb.KV8Cache(k, k, e.int(), e)


def test_every_kv8_name_is_exported():
    import lowbit_b200 as lb
    for n in ("KV8Cache", "kv8_append", "kv8_attention", "kv8_read"):
        assert n in lb.__all__ and callable(getattr(lb, n))
    with pytest.raises(AttributeError):
        lb.kv8_nothing


def test_scale_byte_of_the_oracle():
    assert R.scale_byte(0.0) == 0 and R.scale_byte(127.0) == 127 and R.scale_byte(np.nextafter(127.0, 200)) == 128
    assert R.scale_byte(float(np.finfo(np.float32).max)) == 249 and R.scale_byte(math.inf) == 255
    assert R.scale_byte(1e-45) == 0 and R.scale_byte(63.5) == 126


@pytest.mark.parametrize("cut", [1, 7, 16, 30])
def test_oracle_append_in_pieces_grows_only_the_step(cut):
    """Pieces give the same exponents as one call, and codes at most one step apart
    (older codes are rounded once more when their block's step grows)."""
    rng = np.random.default_rng(cut)
    x = rng.standard_normal((40, (2 + 2) * 32)).astype(np.float32) * np.exp(rng.standard_normal((40, 1))).astype(np.float32)
    ang = np.arange(64)[:, None] * 0.1 ** np.arange(16)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    table = np.array([[2, 0, 1]])

    def empty():
        return {n: np.zeros((3, 1, 16, 32) if len(n) == 1 else (3, 1), np.int8 if len(n) == 1 else np.uint8)
                for n in ("k", "v", "k_exp", "v_exp")}
    one, two = empty(), empty()
    q = R.append(one, x, table, [0], cos, sin, 2)
    q2 = np.concatenate([R.append(two, x[:cut], table, [0], cos, sin, 2), R.append(two, x[cut:], table, [cut], cos, sin, 2)])
    np.testing.assert_array_equal(q, q2)
    for n in ("k", "v"):
        np.testing.assert_array_equal(one[n + "_exp"], two[n + "_exp"])
        assert np.abs(one[n].astype(int) - two[n]).max() <= 1


def test_names_import_without_torch():
    """The package, all its exported names included, does not need torch before it is used."""
    import subprocess
    import sys
    from pathlib import Path
    code = "import sys; sys.modules['torch'] = None\nfrom lowbit_b200 import *\nassert callable(kv8_append) and callable(KV8Cache)"
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parents[1], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_torch_module_builds_without_nvcc(monkeypatch, tmp_path):
    """With a prebuilt library and no nvcc the torch side still builds (it needs CUDA's headers only), or is prebuilt too."""
    from lowbit_b200 import _build
    cxx = tmp_path / "cxx"
    cxx.write_text('#!/bin/sh\necho "$@" > "$0.args"\nwhile [ "$1" != -o ]; do shift; done\ntouch "$2"\n')
    cxx.chmod(0o755)

    def none():
        raise RuntimeError("nvcc not found; set NVCC or CUDA_HOME")
    monkeypatch.setattr(_build, "nvcc", none)
    monkeypatch.setattr(_build, "TORCH_LIB", tmp_path / "_kv8_torch.so")
    monkeypatch.setattr(_build, "TORCH_STAMP", tmp_path / "stamp")
    monkeypatch.setenv("LOWBIT_B200_LIB", str(tmp_path / "lib.so"))
    monkeypatch.setenv("CXX", str(cxx))
    assert _build.build() == tmp_path / "lib.so"
    assert _build.build_torch() == tmp_path / "_kv8_torch.so" and (tmp_path / "_kv8_torch.so").exists()
    assert str(_build.cuda_include()) in (tmp_path / "cxx.args").read_text()
    monkeypatch.setenv("CUDA_HOME", str(tmp_path))
    monkeypatch.setattr(_build.sys, "path", [])
    with pytest.raises(RuntimeError, match="LOWBIT_B200_TORCH_LIB"):
        _build.cuda_include()
    monkeypatch.setenv("LOWBIT_B200_TORCH_LIB", str(tmp_path / "mine.so"))
    assert _build.build_torch() == tmp_path / "mine.so"


def test_build_command_without_torch():
    """The build command prints the library's path alone, and does not need torch."""
    import subprocess
    import sys
    from pathlib import Path

    from lowbit_b200 import _build
    lib = str(_build.build())
    code = "import runpy, sys; sys.modules['torch'] = None; runpy.run_module('lowbit_b200._build', run_name='__main__')"
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parents[1], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.split() == [lib], r.stderr
