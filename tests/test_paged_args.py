"""The paged-cache library loads without a GPU, exports what include/khq_paged.h
declares, and refuses what it does not take before anything is launched."""
import ctypes
import os
import re
import struct
import subprocess

import pytest
import torch

from khq import _lib, paged
from khq.build import PAGED_LIB_PATH

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "khq_paged.h")
FAKE = 0x10000  # never dereferenced: every call here is refused first


def declared():
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return set(re.findall(r"^\s*(?:const\s+)?(?:long\s+)?\w+\*?\s+\**(khq_\w+)\(", src, flags=re.M))


def test_header_symbols_exported():
    names = declared()
    assert names == set(paged.SIGNATURES)
    paged.lib()
    out = subprocess.run(["nm", "-D", "--defined-only", PAGED_LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert {s for s in exported if not s.startswith("_")} == names


def pages(**over):
    f = dict(k=FAKE, v=FAKE, page=64 * 4 * 256, token=4 * 256, head=256, n_pages=8, page_size=64,
             hkv=4, d=256, dtype=0)
    f.update(over)
    return paged.PAGES_STRUCT.pack(*f.values())


def rows(**over):
    f = dict(q=FAKE, q_out=FAKE, k=FAKE, k_out=0, k_normed=0, v=FAKE, qw=0, kw=0, pos=FAKE,
             slots=FAKE)
    f.update({n: 256 for n in ("qt", "qh", "qot", "qoh", "kt", "kh", "kot", "koh", "knt", "knh",
                               "vt", "vh")})
    f.update(theta=1e7, eps=1e-6, n=4, hq=24, hkv=4, d=256, rot=64, pos0=0, rnd=0, dtype=0)
    f.update(over)
    return paged.ROWS_STRUCT.pack(*f.values())


def queries(**over):
    f = dict(q=FAKE, gate=0, out=FAKE, cu=FAKE, kv=FAKE, table=FAKE, ws=0, ws_bytes=0)
    f.update({n: 256 for n in ("qt", "qh", "gt", "gh", "ot", "oh")})
    f.update(scale=0.0625, n_tok=4, n_seq=2, hq=24, ld=8, max_q=4)
    f.update(over)
    return paged.ATTN_STRUCT.pack(*f.values())


@pytest.mark.parametrize("over", [
    dict(k=0), dict(v=0), dict(k=FAKE + 8), dict(page=64 * 4 * 256 + 4), dict(token=-1024),
    dict(head=257), dict(n_pages=0), dict(page_size=0), dict(hkv=0), dict(d=96), dict(dtype=2),
    dict(n_pages=1 << 20, page_size=1 << 12)])
def test_pages_refused(over):
    lib = paged.lib()
    assert lib.khq_paged_attn(queries(), pages(**over), None) == -100
    assert lib.khq_qk_norm_rope(rows(hkv=over.get("hkv", 4), d=over.get("d", 256),
                                     dtype=over.get("dtype", 0)), pages(**over), None) == -100


@pytest.mark.parametrize("over", [
    dict(q=0), dict(out=0), dict(cu=0), dict(kv=0), dict(table=0), dict(ld=0), dict(n_tok=-1),
    dict(n_seq=0), dict(n_seq=4097), dict(hq=0), dict(hq=22), dict(max_q=0), dict(ld=1 << 26)])
def test_attn_refused(over):
    assert paged.lib().khq_paged_attn(queries(**over), pages(), None) == -100


@pytest.mark.parametrize("over", [
    dict(scale=float("inf")), dict(scale=float("nan")), dict(n_tok=1 << 23, hq=16),
    dict(n_seq=4096, hq=1024, hkv=1024)])
def test_attn_sizes_refused(over):
    over = dict(over)
    p = pages(hkv=over.pop("hkv", 4), n_pages=1)
    assert paged.lib().khq_paged_attn(queries(**over), p, None) == -100


@pytest.mark.parametrize("over", [dict(page=0), dict(token=0), dict(head=0), dict(head=128)])
def test_rows_refuse_slots_that_share_memory(over):
    assert paged.lib().khq_qk_norm_rope(rows(), pages(**over), None) == -100


@pytest.mark.parametrize("theta", [float("inf"), -1.0])
def test_rows_theta_refused(theta):
    assert paged.lib().khq_qk_norm_rope(rows(theta=theta), pages(), None) == -100


def test_attn_workspace_refused():
    need = paged.attn_ws_bytes(4, 2, 24, 4, 256, 4)
    lib = paged.lib()
    if need:
        assert lib.khq_paged_attn(queries(ws=FAKE, ws_bytes=need - 1), pages(), None) == -101
        assert lib.khq_paged_attn(queries(ws=FAKE + 4, ws_bytes=need), pages(), None) == -101
    assert lib.khq_paged_attn_ws_bytes(4, 2, 24, 5, 256, 4) == -100
    with pytest.raises(_lib.KhqError):
        paged.attn_ws_bytes(4, 0, 24, 4, 256, 4)


@pytest.mark.parametrize("over", [
    dict(q=0, k=0), dict(q_out=0), dict(hq=0), dict(hkv=0), dict(n=-1), dict(d=32), dict(dtype=3),
    dict(eps=-1.0), dict(eps=float("nan")), dict(rot=63), dict(rot=8), dict(rot=272), dict(rot=-16),
    dict(theta=0.0), dict(theta=float("nan")), dict(pos0=-1), dict(v=0), dict(slots=0)])
def test_rows_refused(over):
    assert paged.lib().khq_qk_norm_rope(rows(**over), pages(), None) == -100


def test_rows_positions_past_32_bits_refused():
    assert paged.lib().khq_qk_norm_rope(rows(pos=0, n=4, pos0=0x7fffffff - 3), pages(), None) == -100


def test_rows_need_somewhere_to_go():
    assert paged.lib().khq_qk_norm_rope(rows(), None, None) == -100
    assert paged.lib().khq_qk_norm_rope(rows(hkv=8), pages(), None) == -100
    assert paged.lib().khq_qk_norm_rope(rows(dtype=1), pages(), None) == -100
    assert paged.lib().khq_qk_norm_rope(None, pages(), None) == -100


@pytest.mark.parametrize("over", [
    {i: None} for i in (0, 1, 2, 4, 5, 10, 11, 12, 13, 14, 15, 16)] + [
    {3: 0}, {6: 0}, {6: 4097}, {7: 0}, {8: 0}, {9: -1}, {7: 1 << 20, 8: 1 << 12}, {3: 1 << 26, 8: 64}])
def test_plan_refused(over):
    args = [FAKE, FAKE, FAKE, 8, FAKE, FAKE, 2, 16, 64, 4] + [FAKE] * 7 + [None]
    for i, x in over.items():
        args[i] = x
    assert paged.lib().khq_paged_plan(*args) == -100


def test_struct_sizes():
    assert (paged.PAGES_STRUCT.size, paged.ROWS_STRUCT.size, paged.ATTN_STRUCT.size) == (64, 224, 136)
    assert struct.calcsize("P") == ctypes.sizeof(ctypes.c_void_p) == 8


def test_host_tensors_refused():
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        paged.plan(z, z, z, z, z, page_size=4, cu_q=z, seq_kv=z, kv_out=z, state_out=z, status=z,
                   positions=z, slots=z)
    x = torch.zeros((1, 4, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        paged.qk_norm_rope(x, None, x)
    with pytest.raises(ValueError, match="device tensor"):
        paged.attn(x, x, x, x, cu_q=z, seq_kv=z, table=z, max_q=1, scale=1.0)
    with pytest.raises(ValueError):
        paged.PageTable(0, 1, 1, 1, 1, device="cpu")


def test_overlapping_outputs_refused():
    x = torch.zeros((4, 64), dtype=torch.float16)
    for t in (x[:, None].expand(4, 3, 64), x[None].expand(2, 4, 64),
              x.as_strided((3, 2, 64), (32, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            paged._written((0, *t.stride()[:2]), t.shape, "out")
    for t in (torch.zeros(4, 3, 64), torch.zeros(3, 4, 64).transpose(0, 1), torch.zeros(1, 1, 64),
              torch.zeros(4, 3, 128)[..., :64], torch.zeros(0, 3, 64)):
        paged._written((0, *t.stride()[:2]), t.shape, "out")
