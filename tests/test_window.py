"""The windowed attention node's C ABI: what the library exports and what it refuses, on the host."""
from __future__ import annotations

import ctypes

import pytest

from strataflow_amd import _lib
from strataflow_amd.paged_kv import rope_desc

from .test_abi import INCLUDE, declared_symbols, desc

OK, BAD, UNS = _lib.SFA_OK, _lib.SFA_ERR_INVALID_ARGUMENT, _lib.SFA_ERR_UNSUPPORTED
P = 0x1000  # never dereferenced
MAX = 2**31 - 1


def test_header_matches_binding_list():
    names = declared_symbols(INCLUDE / "sfa_window.h")
    assert names == set(_lib.WINDOW_EXPORTS)
    lib = _lib.load()
    for name in names:
        assert hasattr(lib, name), name


def append(kv=None, rope=None, **kw):
    a = dict(q=P, qs=32 * 128, out=2 * P, k=P, ks=8 * 128, v=P, vs=8 * 128, qn=P, kn=P, eps=1e-6, seq=P, pos=P, rp=None, n=2,
             table=P, mp=4)
    a.update(kw)
    return _lib.load().sfa_norm_rope_kv_append(kv or desc(), rope or rope_desc(128, 1e4), a["q"], a["qs"], a["out"], a["k"], a["ks"],
                                               a["v"], a["vs"], a["qn"], a["kn"], a["eps"], a["seq"], a["pos"], a["rp"], a["n"],
                                               a["table"], a["mp"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), OK), (dict(n=-1), BAD), (dict(mp=0), BAD), (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD),
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(seq=None), BAD), (dict(pos=None), BAD), (dict(table=None), BAD),
    (dict(q=None), BAD), (dict(out=None), BAD),               # q without q_out and the other way round
    (dict(qs=32 * 128 - 4), BAD), (dict(ks=8 * 128 - 4), BAD), (dict(vs=0), BAD),
    (dict(qs=32 * 128 + 2), UNS), (dict(ks=8 * 128 + 1), UNS), (dict(vs=8 * 128 + 3), UNS),
    (dict(out=P, qs=48 * 128), BAD),                            # in place on rows with a stride
    (dict(q=P + 4), UNS), (dict(out=P + 8), UNS), (dict(k=P + 4), UNS), (dict(v=P + 4), UNS),
])
def test_append_refusals(kw, want):
    assert append(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(n_rot=0), BAD), (dict(n_rot=136), BAD), (dict(n_rot=12), UNS), (dict(pairing=1), BAD), (dict(freq_base=0.0), BAD),
    (dict(freq_base=float("inf")), BAD), (dict(freq_base=float("nan")), BAD), (dict(n_axis=0), BAD), (dict(n_axis=5), BAD),
    (dict(n_axis=3, sections=(20, 20, 20)), BAD), (dict(n_axis=2, sections=(-1, 65)), BAD), (dict(n_axis=2, sections=(32, 32), layout=7), BAD),
    (dict(n_axis=2, sections=(31, 33), layout=1), BAD),         # 33 pairs of axis 1 are not there to be dealt
    (dict(n_axis=2, sections=(32, 32), layout=1), OK), (dict(n_axis=3, sections=(0, 64, 0)), OK), (dict(n_rot=8), OK),
])
def test_rope_refusals(kw, want):
    r = rope_desc(128, 1e4)
    for name, v in kw.items():
        if name == "sections":
            r.sections[:len(v)] = v
        else:
            setattr(r, name, v)
    assert _lib.load().sfa_rope_desc_check(ctypes.byref(r), 128) == want
    if want != OK:
        assert append(rope=r) == want


def test_rope_check_without_a_rotation():
    assert _lib.load().sfa_rope_desc_check(None, 128) == BAD


def decode(kv=None, **kw):
    a = dict(q=P, out=P, table=P, mp=4, lens=P, window=64, sink=4, B=2, most=500, scale=0.1, ws=P, size=1 << 30)
    a.update(kw)
    return _lib.load().sfa_attn_decode_window(kv or desc(), a["q"], a["out"], a["table"], a["mp"], a["lens"], a["window"], a["sink"], a["B"],
                                              a["most"], a["scale"], a["ws"], a["size"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(B=0), OK), (dict(B=-1), BAD), (dict(q=None), BAD), (dict(out=None), BAD), (dict(table=None), BAD), (dict(lens=None), BAD),
    (dict(mp=0), BAD), (dict(window=0), BAD), (dict(window=-3), BAD), (dict(sink=-1), BAD), (dict(most=0), BAD), (dict(scale=0.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(ws=None), BAD), (dict(size=0), BAD), (dict(ws=P + 16), UNS),
    (dict(q=P + 4), UNS), (dict(out=P + 4), UNS),
])
def test_decode_refusals(kw, want):
    assert decode(**kw) == want


def prefill(kv=None, **kw):
    a = dict(q=P, out=P, table=P, mp=4, pos0=0, T=5, window=64, sink=4, scale=0.1, ws=P, size=1 << 30)
    a.update(kw)
    return _lib.load().sfa_attn_prefill_window(kv or desc(), a["q"], a["out"], a["table"], a["mp"], a["pos0"], a["T"], a["window"], a["sink"],
                                               a["scale"], a["ws"], a["size"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(T=0), OK), (dict(T=-1), BAD), (dict(pos0=-1), BAD), (dict(pos0=MAX, T=1), BAD), (dict(q=None), BAD), (dict(out=None), BAD),
    (dict(table=None), BAD), (dict(mp=0), BAD), (dict(window=0), BAD), (dict(sink=-1), BAD), (dict(scale=-1.0), BAD),
    (dict(q=P + 4), UNS), (dict(out=P + 4), UNS),
])
def test_prefill_refusals(kw, want):
    assert prefill(**kw) == want


def test_descriptor_refusals():
    for kv, want in ((desc(head_dim=96), UNS), (desc(n_head=24), UNS), (desc(n_head=30), BAD), (desc(page_size=40), BAD),
                     (desc(kv_type=_lib.SFA_KV_Q8_0, head_dim=32), UNS), (desc(kv_type=2), UNS)):
        assert decode(kv=kv) == want and prefill(kv=kv) == want and append(kv=kv) == want
    assert prefill(kv=desc(page_size=32)) == UNS
    assert decode(kv=desc(page_size=32), B=0) == OK


def test_limits_of_a_launch():
    """What a grid or a 32-bit offset cannot hold is refused, not cut."""
    size = 1 << 44
    many = desc(n_head=1, n_head_kv=1)
    assert decode(kv=many, B=65536, size=size) == UNS
    assert prefill(kv=many, T=65535 * 128 + 1, size=size) == UNS
    wide = desc(kv_type=_lib.SFA_KV_F32, head_dim=128, n_head=32769, n_head_kv=32769, page_size=64)
    assert decode(kv=wide, size=size) == UNS and prefill(kv=wide, size=size) == UNS
    assert decode(scale=3e38) == BAD and prefill(scale=3e38) == BAD  # times log2(e) it is no f32


def test_workspace_sizes():
    lib = _lib.load()
    for bad in ((0, 500, 64, 4), (2, 0, 64, 4), (2, 500, 0, 4), (2, 500, 64, -1)):
        assert lib.sfa_decode_window_workspace_bytes(desc(), *bad) == 0
    need = lib.sfa_decode_window_workspace_bytes(desc(), 2, 500, 64, 4)
    assert need > 0 and decode(size=need - 1) == BAD
    # a call's need does not grow with what it cannot attend
    assert lib.sfa_decode_window_workspace_bytes(desc(), 2, MAX, 64, 4) <= lib.sfa_decode_window_workspace_bytes(desc(), 2, MAX, MAX, MAX) < 1 << 30
    for bad in ((-1, 5, 64, 4), (0, 0, 64, 4), (0, 5, 0, 4), (0, 5, 64, -1), (MAX, 5, 64, 4)):
        assert lib.sfa_prefill_window_workspace_bytes(desc(), *bad) == 0
    # the bound covers every call of up to so many tokens
    import random
    rng = random.Random(0)
    for _ in range(3000):
        g = rng.choice([1, 2, 4, 8])
        hkv = rng.choice([1, 2, 3, 8, 16, 64])
        kv = desc(n_head=g * hkv, n_head_kv=hkv, kv_type=rng.choice([0, 1, 8]), head_dim=rng.choice([64, 128]))
        T = rng.randint(1, rng.choice([4, 64, 1000, 9000]))
        need = lib.sfa_prefill_window_workspace_bytes(kv, rng.randint(0, 100000), T, rng.randint(1, 20000), rng.randint(0, 300))
        assert need <= lib.sfa_prefill_window_workspace_bound(kv, T)
        assert lib.sfa_prefill_window_workspace_bound(kv, T) <= lib.sfa_prefill_window_workspace_bound(kv, T + 77)
    assert lib.sfa_prefill_window_workspace_bound(desc(), 0) == 0


def test_prefill_needs_its_workspace():
    need = _lib.load().sfa_prefill_window_workspace_bytes(desc(), 20000, 93, 4096, 4)
    assert need > 0
    assert prefill(pos0=20000, T=93, window=4096, ws=None) == BAD
    assert prefill(pos0=20000, T=93, window=4096, size=need - 1) == BAD
    assert prefill(pos0=20000, T=93, window=4096, ws=P + 64) == UNS


def test_rows_past_32_bit_tiles_are_refused():
    assert decode(kv=desc(n_head=1 << 20, n_head_kv=1 << 20)) == UNS
    assert prefill(kv=desc(n_head=1 << 20, n_head_kv=1 << 20)) == UNS


def test_python_refusals():
    """What the wrapper checks before a pointer is passed on (on the host: tensors without a GPU)."""
    import torch

    from strataflow_amd.paged_kv import PagedKV
    kv = PagedKV(1, 8, 2, 64, _lib.SFA_KV_F16, 64, 2, device="cpu")
    q, i = torch.zeros(2, 8, 64), torch.zeros(2, dtype=torch.int32)
    for bad in (q.double(), q[:, :4], q.transpose(0, 1).contiguous(), torch.zeros(2, 8, 128)[..., :64]):
        with pytest.raises(ValueError):
            kv._rows(bad, None, 2, None)
    with pytest.raises(ValueError):
        kv._rows(q, torch.zeros(2, 511), 2, None)
    x = torch.zeros(2, 12, 64)
    assert kv._heads(x[:, 8:10], "k", 2, 2) == 12 * 64
    for bad in (x[:, 8:10].double(), x[:, 8:11], x[:, ::6], x.transpose(0, 1)[:2, :2]):
        with pytest.raises(ValueError):
            kv._heads(bad, "k", 2, 2)
    assert i.numel() == 2


def test_pager_create_refusals():
    lib = _lib.load_host()
    c = _lib.SfaPagerConfig(1, 8, 2, 64, _lib.SFA_KV_F16, 64, 1, 256, 128, _lib.SFA_ATTEND_WINDOW, 0, 0, 0)
    h = ctypes.c_void_p(1)

    def create(n_sink, **kw):
        d = _lib.SfaPagerConfig.from_buffer_copy(c)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.sfa_pager_create_sinks(ctypes.byref(d), n_sink, ctypes.byref(h))

    assert create(-1) == BAD and h.value is None
    assert create(4, attend=_lib.SFA_ATTEND_LOSSLESS) == BAD
    assert create(4, window=0) == BAD
    assert create(4, page_size=96) == UNS
    assert lib.sfa_pager_create_sinks(None, 4, ctypes.byref(h)) == BAD
    assert lib.sfa_pager_create_sinks(ctypes.byref(c), 4, None) == BAD
    assert lib.sfa_pager_norm_rope_append(None, 0, None, None, 0, None, None, 0, None, 0, None, None, 1e-6, None, None) == BAD


def test_page_planner_sinks_cpp(tmp_path):
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    host, exe = root / "strataflow_amd" / "host", tmp_path / "page_planner_sinks_test"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{host}", str(root / "tests" / "cpp" / "page_planner_sinks_test.cpp"),
                    str(host / "page_planner.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert out.startswith("ok ") and int(out.split()[1]) > 1000
