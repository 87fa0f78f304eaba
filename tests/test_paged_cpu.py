"""Host side of the paged K/V cache operators: argument checks of the C ABI and
of the Python entry points (no kernel launches), and the tests' plain forms
against the oracle."""

import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import oracle
from hspmn_b200 import _native as N
from hspmn_b200 import ops
from tests import paged_ref as ref
from tests.conftest import PKG

P = ctypes.c_void_p(4096)
INVALID, DTYPE, ALIGN, UNSUPPORTED = -1, -2, -3, -4


def test_slots_refusals():
    def slots(table=P, rs=8, seq=P, new=P, free=P, nfree=4, R=2, Pw=8, page=16, n=4, cu=P, kv=P, pos=P, out=P, taken=P):
        return N.lib().hspmn_paged_slots(table, rs, seq, new, free, nfree, R, Pw, page, n, cu, kv, pos, out, taken, None)

    for over in (dict(table=None), dict(seq=None), dict(new=None), dict(free=None), dict(cu=None), dict(kv=None),
                 dict(pos=None), dict(out=None), dict(taken=None), dict(rs=7), dict(R=-1), dict(n=-1), dict(nfree=-1),
                 dict(Pw=-1), dict(n=1 << 31), dict(R=8192, Pw=1 << 19, rs=1 << 19)):
        assert slots(**over) == INVALID, over
    for over in (dict(page=0), dict(page=4), dict(page=24), dict(page=8192), dict(R=8193)):
        assert slots(**over) == UNSUPPORTED, over


def test_write_refusals():
    def write(k=P, sn=512, sh=128, v=P, cos=P, sin=P, ts=128, rows=9, tdt=2, pos=P, slots=P, kc=P, sp=8192, ss=512, vc=P,
              n=3, heads=4, hd=128, pages=5, page=16, dt=2):
        return N.lib().hspmn_rope_paged_write(k, sn, sh, v, sn, sh, cos, sin, ts, rows, tdt, pos, slots, kc, sp, ss, sh,
                                              vc, sp, ss, sh, n, heads, hd, pages, page, dt, None)

    for over in (dict(k=None), dict(v=None), dict(sin=None), dict(cos=None), dict(pos=None), dict(slots=None),
                 dict(kc=None), dict(vc=None), dict(n=-1), dict(heads=0), dict(ts=127), dict(rows=-1), dict(sn=-512)):
        assert write(**over) == INVALID, over
    for over in (dict(dt=9), dict(tdt=1)):
        assert write(**over) == DTYPE, over
    for over in (dict(page=12), dict(hd=24, ts=24), dict(hd=12, cos=None, sin=None)):
        assert write(**over) == UNSUPPORTED, over
    odd = ctypes.c_void_p(4104)
    for over in (dict(k=odd), dict(v=odd), dict(cos=odd), dict(kc=odd), dict(vc=odd), dict(sn=516), dict(ss=516),
                 dict(ts=132)):
        assert write(**over) == ALIGN, over
    assert write(n=0) == 0 and write(n=0, k=None) == 0


def test_attention_refusals():
    def fwd(q=P, sn=2048, sh=128, kc=P, sp=8192, ss=512, vc=P, table=P, rs=8, kv=P, cu=P, pos=P, o=P, n=3, R=2, Pw=8,
            pages=5, page=16, H=16, Hkv=4, hd=128, dt=2, scale=0.1, max_q=0, ws=P, wsb=1 << 30):
        return N.lib().hspmn_sqdk_paged_fwd(q, sn, sh, kc, sp, ss, sh, vc, sp, ss, sh, table, rs, kv, cu, pos, o, sn, sh,
                                            n, R, Pw, pages, page, H, Hkv, hd, dt, scale, max_q, ws, wsb, None)

    for over in (dict(q=None), dict(o=None), dict(kc=None), dict(vc=None), dict(table=None), dict(kv=None), dict(cu=None),
                 dict(pos=None), dict(n=-1), dict(R=-1), dict(rs=7), dict(scale=0.0), dict(scale=float("nan")),
                 dict(max_q=-1), dict(sn=-2048), dict(n=1 << 28), dict(Pw=1 << 28, rs=1 << 28),
                 dict(Pw=(1 << 27) - 255, rs=1 << 28), dict(R=1 << 25)):
        assert fwd(**over) == INVALID, over
    for over in (dict(dt=0), dict(dt=7)):
        assert fwd(**over) == DTYPE, over
    for over in (dict(hd=12), dict(hd=136), dict(H=14), dict(H=516), dict(page=48), dict(sp=1 << 30),
                 dict(ss=1 << 28)):
        assert fwd(**over) == UNSUPPORTED, over
    odd = ctypes.c_void_p(4104)
    for over in (dict(q=odd), dict(o=odd), dict(kc=odd), dict(vc=odd), dict(ws=odd), dict(sn=2052), dict(ss=516)):
        assert fwd(**over) == ALIGN, over
    assert fwd(n=0) == 0 and fwd(n=0, q=None) == 0


def test_ops_refuse_cpu_tensors():
    t, i, x = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2, 16))
    c, j = torch.zeros((2, 8, 2, 16)), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.paged_slots_(t, i, i, i, 8, 1)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.rope_paged_write_(x, x, None, None, j, j, c, c)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.sqdk_paged_fwd(x, c, c, t, i, i, j, 0.1)


def python(code, path):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          env=dict(os.environ, PYTHONPATH=str(path), CUDA_VISIBLE_DEVICES=""))


def test_importing_the_package_loads_no_library():
    r = python("import hspmn_b200, torch\n"
               "from hspmn_b200 import HSPMNBlock, HSPMNConfig\n"
               "HSPMNBlock(HSPMNConfig(dim=64, num_heads=4, num_kv_heads=2))\n"
               "for name in ('paged_slots_', 'rope_paged_write_', 'sqdk_paged_fwd'):\n"
               "    getattr(torch.ops.hspmn, name).default\n"
               "assert 'libhspmn' not in open('/proc/self/maps').read()\n"
               "t = torch.zeros((1, 2), dtype=torch.int32)\n"
               "for op in (hspmn_b200.ops.paged_slots_, torch.ops.hspmn.paged_slots_):\n"
               "    try:\n"
               "        op(t, t[0, :1], t[0, :1], t[0], 8, 1)\n"
               "        assert False\n"
               "    except RuntimeError as e:\n"
               "        assert 'CUDA tensors' in str(e), e\n"
               "assert 'libhspmn_torch' in open('/proc/self/maps').read()\n", PKG)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("torch_lib", [None, b"built for something else"])
def test_package_without_a_fitting_operator_library(tmp_path, torch_lib):
    """The rest of the package works; a paged operator says what to do, called or registered."""
    pkg = tmp_path / "hspmn_b200"
    pkg.mkdir()
    for f in os.listdir(os.path.dirname(N.LIB_PATH)):
        if f.endswith(".py") or f == N.LIB_NAME:
            os.symlink(os.path.join(os.path.dirname(N.LIB_PATH), f), pkg / f)
    if torch_lib is not None:
        (pkg / os.path.basename(N.TORCH_LIB_PATH)).write_bytes(torch_lib)
    r = python("import hspmn_b200, torch\n"
               f"assert hspmn_b200.__file__.startswith({str(tmp_path)!r})\n"
               "assert hspmn_b200.native_available() and hspmn_b200._native.lib().hspmn_version() > 0\n"
               "t = torch.zeros((1, 2), dtype=torch.int32)\n"
               "for op in (hspmn_b200.ops.paged_slots_, torch.ops.hspmn.paged_slots_):\n"
               "    for _ in range(2):\n"
               "        try:\n"
               "            op(t, t[0, :1], t[0, :1], t[0], 8, 1)\n"
               "            assert False\n"
               "        except RuntimeError as e:\n"
               "            assert 'build_native.py' in str(e), e\n", tmp_path)
    assert r.returncode == 0, r.stderr[-2000:]


def test_operator_library_is_rebuilt_for_another_pytorch(tmp_path, monkeypatch):
    """A file newer than its sources does not do: it must be built for this PyTorch and Python."""
    import build_native
    assert build_native.torch_ops_up_to_date()  # as built
    lib = tmp_path / "libhspmn_torch.so"
    monkeypatch.setattr(build_native, "TORCH_LIB", str(lib))
    assert not build_native.torch_ops_up_to_date()
    with open(N.TORCH_LIB_PATH, "rb") as f:
        built = f.read()
    mark = N.torch_build_id().encode()
    assert built.count(mark) == 1 and torch.__version__.encode() in mark
    lib.write_bytes(built)
    assert build_native.torch_ops_up_to_date()
    lib.write_bytes(built.replace(mark, mark.replace(torch.__version__.encode(), b"x" * len(torch.__version__))))
    assert not build_native.torch_ops_up_to_date()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    lib.write_bytes(built)
    assert not build_native.torch_ops_up_to_date()
    # and is not loaded: entry points may have changed their meaning without changing their names
    monkeypatch.setattr(N, "TORCH_LIB_PATH", str(lib))
    with pytest.raises(RuntimeError, match="build_native.py"):
        N.load_torch_ops()


def test_cuda_library_is_built_without_the_operator_library(monkeypatch):
    """A host without PyTorch or with another compiler still gets the library of the C ABI, and is told."""
    import build_native

    def fails(*args):
        raise RuntimeError("g++ failed: no such header")

    monkeypatch.setattr(build_native, "build_torch_ops", fails)
    with pytest.warns(RuntimeWarning, match="paged-cache operators.*no such header"):
        assert build_native.build() == build_native.LIB
    monkeypatch.setattr(build_native, "run", fails)  # the CUDA library itself must build
    with pytest.raises(RuntimeError, match="g.. failed"):
        build_native.build(force=True)


def test_dependent_kernels_wait_before_they_release():
    """A kernel that let the next one begin in front of its own wait would let the 16-row attention kernel, which
    counts on the wait of the kernel before it, read what is still being written."""
    import build_native
    text = {os.path.basename(f): open(f).read() for f in build_native.sources() if f.endswith((".cu", ".cuh"))}
    begins = ("grid_dependency_enter();", "grid_dependency_behind();")
    kernels = 0
    for name in ("paged.cuh", "paged_attn.cuh", "paged_chunk.cuh"):
        assert "grid_dependents_launch" not in text[name] and "griddepcontrol" not in text[name], name
        for body in text[name].split("__global__")[1:]:
            kernels += 1
            assert begins[0] in body, name
    assert kernels == 6
    assert sum(t.count(begins[1]) for n, t in text.items() if n != "common.cuh") == 1
    enter = text["common.cuh"].split("void grid_dependency_enter() {")[1].split("}")[0]
    assert enter.index("grid_dependency_wait();") < enter.index("grid_dependents_launch();")


def test_plain_attention_is_the_oracles():
    g = torch.Generator().manual_seed(0)
    B, S, H, Hkv, hd, page = 2, 45, 6, 2, 16, 8
    k, v = torch.randn((B, 48, Hkv, hd), generator=g), torch.randn((B, 48, Hkv, hd), generator=g)
    idx = torch.stack([torch.randperm(S, generator=g)[:9].sort().values for _ in range(B)])
    q = torch.randn((B, 9, H, hd), generator=g)
    want = oracle.sqdk_fp32(q.numpy(), k[:, :S].numpy(), v[:, :S].numpy(), idx.numpy())
    order = torch.randperm(12, generator=g)
    kc, vc = torch.empty((12, page, Hkv, hd)), torch.empty((12, page, Hkv, hd))
    kc[order], vc[order] = k.reshape(12, page, Hkv, hd), v.reshape(12, page, Hkv, hd)
    got, _ = ref.attend_ref(q.reshape(-1, H, hd).half(), kc, vc, order.view(B, 6), [S, S], [0, 9, 18], idx.reshape(-1),
                            hd ** -0.5)
    got32, _ = ref.attend_ref(q.reshape(-1, H, hd), kc, vc, order.view(B, 6), [S, S], [0, 9, 18], idx.reshape(-1), hd ** -0.5)
    np.testing.assert_allclose(got32.numpy().reshape(want.shape), want, atol=2e-5)
    assert got.dtype == torch.float64


def test_plain_slots():
    table, cu, kv, pos, slots, taken = ref.slots_ref([[7, -1], [3, 4]], [6, 16], [4, 0], [9, 2], 8, 5)
    assert table == [[7, 9], [3, 4]] and cu == [0, 4, 4] and kv == [10, 16] and taken == 1
    assert pos == [6, 7, 8, 9, -1] and slots == [62, 63, 72, 73, -1]
