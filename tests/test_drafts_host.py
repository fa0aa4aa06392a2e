"""The C ABI, Python layer and oracle of the operators of drafted tokens without a GPU: the header and its ctypes mirror
agree, calls that cannot be right are refused on the host, and oracle/drafts.py matches independent forms."""
from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

import bsa_mi355x as bsa
from bsa_mi355x import _lib, drafts, serving
from oracle import drafts as dft
from oracle import serving as orc
from test_codegen import _device_asm, _functions
from test_serving_host import BAD_CACHES, FAKE, _cache, _pool

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "bsgdraft.h")
UNITS = ("kv_rotate.hip", "kv_tree.hip", "verify.hip", "pages_keep.hip")


def test_header_and_library_agree(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(bsg_[a-z0-9_]+)\s*\(", text))
    assert len(names) == 7
    lib = bsa.load()
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES, name
        declared = re.search(name + r"\s*\((.*?)\);", text, re.S).group(1)
        assert len(declared.split(",")) == len(_lib.SIGNATURES[name][1]), name
    assert drafts.MAX_NODES == int(re.search(r"BSG_TREE_NODES (\d+)", text).group(1))
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("gcc not available")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    prints = 'printf("%zu\\n", sizeof(bsg_rotary));' + "".join(f'printf("%zu\\n", offsetof(bsg_rotary, {f}));' for f, _ in _lib.Rotary._fields_)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "bsgdraft.h"\nint main(void){' + prints + "return 0;}")
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()))
    assert got == [ctypes.sizeof(_lib.Rotary)] + [getattr(_lib.Rotary, f).offset for f, _ in _lib.Rotary._fields_]


def _rotary(**kw):
    a = dict(cos=FAKE, sin=FAKE, stride=64, positions=100, dims=128, interleaved=0, eps=1e-6, q_norm=None, k_norm=None,
             token_positions=None, parents=None)
    a.update(kw)
    return _lib.Rotary(*a.values())


def _append(cache, rotary=None, q=FAKE, qs=(512, 128), heads=4, out=FAKE, os_=(512, 128), k=FAKE, tokens=4, rows=4, cu=None, max_new=1,
            dtype=0, slots=None):
    return bsa.load().bsg_kv_append_rotated(q, *qs, heads, out, *os_, k, 256, 128, FAKE, 256, 128, tokens, rotary or _rotary(),
                                            cache, slots, rows, cu, max_new, dtype, None)


def _attend(cache, q=FAKE, qs=(512, 128), tokens=4, heads=4, parents=FAKE, rows=4, cu=None, max_new=1, max_len=0, scale=0.1, out=FAKE,
            os_=(512, 128), dtype=0, ws=FAKE, ws_bytes=1 << 40, cus=256, slots=None):
    return bsa.load().bsg_kv_tree_attention(q, *qs, tokens, heads, parents, ctypes.byref(cache), slots, rows, cu, max_new, max_len, scale,
                                            out, *os_, None, dtype, ws, ws_bytes, cus, None)


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_bad_caches_are_refused(bad, code):
    assert _append(_cache(**bad)) == code
    assert _attend(_cache(**bad)) == code
    assert bsa.load().bsg_kv_tree_attention_workspace_bytes(ctypes.byref(_cache(**bad)), 4, 4, 1, 0, 256) == -1
    assert _lib.last_error()


def test_bad_rotations_are_refused():
    c = _cache()
    for bad, code in ((dict(cos=None), _lib.BSG_ERR_ARG), (dict(sin=None), _lib.BSG_ERR_ARG), (dict(dims=24), _lib.BSG_ERR_UNSUPPORTED),
                      (dict(dims=256), _lib.BSG_ERR_UNSUPPORTED), (dict(positions=0), _lib.BSG_ERR_ARG), (dict(stride=60), _lib.BSG_ERR_ARG),
                      (dict(eps=-1.0), _lib.BSG_ERR_ARG), (dict(eps=float("nan")), _lib.BSG_ERR_ARG), (dict(cos=FAKE + 4), _lib.BSG_ERR_ALIGN),
                      (dict(stride=66), _lib.BSG_ERR_ALIGN), (dict(q_norm=FAKE + 2), _lib.BSG_ERR_ALIGN),
                      (dict(token_positions=FAKE, parents=FAKE), _lib.BSG_ERR_ARG)):
        assert _append(c, _rotary(**bad)) == code, bad
    assert _append(_cache(head_dim=64), _rotary(dims=128)) == _lib.BSG_ERR_ARG
    assert _append(c, _rotary(parents=FAKE), cu=FAKE, max_new=65) == _lib.BSG_ERR_UNSUPPORTED
    assert _append(c, heads=0) == _lib.BSG_ERR_ARG
    assert _append(c, q=None) == _lib.BSG_ERR_ARG
    assert _append(c, k=None) == _lib.BSG_ERR_ARG
    assert _append(c, k=FAKE + 1) == _lib.BSG_ERR_ALIGN
    assert _append(c, q=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert _append(c, out=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert _append(c, qs=(516, 128)) == _lib.BSG_ERR_ALIGN
    assert _append(c, os_=(512, 132)) == _lib.BSG_ERR_ALIGN
    assert _append(c, dtype=2) == _lib.BSG_ERR_DTYPE
    assert _append(c, tokens=5) == _lib.BSG_ERR_ARG
    assert _append(c, rows=5, tokens=5) == _lib.BSG_ERR_ARG
    assert _append(c, tokens=0, rows=0) == 0
    for most in (2 ** 31 - 1, 2 ** 31 - 14):  # counted in 64 bits
        assert _append(c, cu=FAKE, max_new=most) == _lib.BSG_ERR_UNSUPPORTED
    assert bsa.load().bsg_kv_append_rotated(FAKE, 512, 128, 4, FAKE, 512, 128, FAKE, 256, 128, FAKE, 256, 128, 4, None, c, None, 4, None, 1,
                                            0, None) == _lib.BSG_ERR_ARG


def test_bad_trees_are_refused():
    c = _cache()
    assert _attend(c, parents=None) == _lib.BSG_ERR_ARG
    assert _attend(c, heads=3) == _lib.BSG_ERR_ARG
    assert _attend(c, q=None) == _lib.BSG_ERR_ARG
    assert _attend(c, cus=0) == _lib.BSG_ERR_ARG
    assert _attend(c, q=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert _attend(c, out=FAKE + 4) == _lib.BSG_ERR_ALIGN
    assert _attend(c, dtype=2) == _lib.BSG_ERR_DTYPE
    assert _attend(c, scale=float("nan")) == _lib.BSG_ERR_ARG
    assert _attend(c, max_new=65, tokens=260) == _lib.BSG_ERR_UNSUPPORTED
    assert _attend(c, rows=70000, tokens=70000, slots=FAKE) == _lib.BSG_ERR_UNSUPPORTED
    assert _attend(c, max_new=0, tokens=0) == 0
    long = _cache(max_pages=4096, table_stride=4096)
    need = bsa.load().bsg_kv_tree_attention_workspace_bytes(ctypes.byref(long), 4, 4, 1, 0, 256)
    assert need > serving.COUNTER_BYTES
    assert _attend(long, ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert _attend(long, ws=None) == _lib.BSG_ERR_WORKSPACE
    assert _attend(long, ws=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert bsa.load().bsg_kv_tree_attention_workspace_bytes(ctypes.byref(long), 4, 4, 65, 0, 256) == -1


def test_bad_verifications_are_refused():
    lib = bsa.load()

    def call(logits=FAKE, draft=None, tokens=8, vocab=1000, ids=FAKE, u=FAKE, parents=None, cu=None, rows=2, max_new=4, temp=1.0,
             temps=None, accepted=FAKE, path=FAKE, out=FAKE, dtype=0, ws=FAKE, ws_bytes=1 << 30):
        return lib.bsg_verify_drafts(logits, 1000, draft, 1000, tokens, vocab, ids, u, parents, cu, rows, max_new, temp, temps, accepted,
                                     path, out, dtype, ws, ws_bytes, None)

    for bad in (dict(logits=None), dict(ids=None), dict(u=None), dict(accepted=None), dict(path=None), dict(out=None), dict(tokens=7),
                dict(rows=-1), dict(vocab=0), dict(max_new=-1), dict(temp=-1.0), dict(temp=float("nan")), dict(temp=float("inf"))):
        assert call(**bad) == _lib.BSG_ERR_ARG, bad
    assert call(dtype=3) == _lib.BSG_ERR_DTYPE
    assert call(max_new=65, tokens=130) == _lib.BSG_ERR_UNSUPPORTED
    assert call(vocab=(1 << 20) + 1) == _lib.BSG_ERR_UNSUPPORTED
    assert call(rows=16385, cu=FAKE) == _lib.BSG_ERR_UNSUPPORTED
    assert call(draft=FAKE, parents=FAKE) == _lib.BSG_ERR_UNSUPPORTED
    assert call(logits=FAKE + 1) == _lib.BSG_ERR_ALIGN
    assert call(draft=FAKE + 2, dtype=2) == _lib.BSG_ERR_ALIGN
    need = lib.bsg_verify_drafts_workspace_bytes(8, 2, 1000, 4, 0, 0)
    assert need > serving.COUNTER_BYTES and call(ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert lib.bsg_verify_drafts_workspace_bytes(8, 2, 1000, 4, 0, 1) > need
    assert call(ws=None) == _lib.BSG_ERR_WORKSPACE
    assert call(ws=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert call(rows=0, tokens=0) == 0
    assert lib.bsg_verify_drafts_workspace_bytes(8, 2, 0, 4, 0, 0) == -1


def test_a_verification_of_slots_is_one_of_the_others():
    """bsgdraft_slots.h declares what ctypes calls, and its checks are bsg_verify_drafts's, whatever slots are."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "bsgdraft_slots.h")).read(), flags=re.S)
    assert re.findall(r"\b(bsg_[a-z0-9_]+)\s*\(", text) == ["bsg_verify_drafts_slots"]
    declared = re.search(r"bsg_verify_drafts_slots\s*\((.*?)\);", text, re.S).group(1)
    types = _lib.SIGNATURES["bsg_verify_drafts_slots"][1]
    assert len(declared.split(",")) == len(types)
    plain = _lib.SIGNATURES["bsg_verify_drafts"][1]
    assert types[:10] + types[11:] == plain and declared.split(",")[10].split() == ["const", "int32_t*", "slots"]
    args = [FAKE, 1000, None, 1000, 8, 1000, FAKE, FAKE, None, None, FAKE, 2, 4, 1.0, None, FAKE, FAKE, FAKE, 0, FAKE, 1 << 30, None]
    lib = bsa.load()
    for i, bad, code in ((0, None, _lib.BSG_ERR_ARG), (4, 7, _lib.BSG_ERR_ARG), (15, None, _lib.BSG_ERR_ARG), (18, 3, _lib.BSG_ERR_DTYPE),
                         (12, 65, _lib.BSG_ERR_ARG), (19, None, _lib.BSG_ERR_WORKSPACE), (20, 64, _lib.BSG_ERR_WORKSPACE)):
        for slots in (FAKE, None):
            call = args[:i] + [bad] + args[i + 1:]
            call[10] = slots
            assert lib.bsg_verify_drafts_slots(*call) == (_lib.BSG_ERR_UNSUPPORTED if bad == 65 else code), (i, slots)
    assert lib.bsg_verify_drafts_slots(*args[:4], 0, *args[5:11], 0, *args[12:]) == 0  # no sequences


def test_documented_last_tokens():
    """The documented line for what the next trees begin with, run as it stands: the new token, or, where nothing was accepted, what
    it was before."""
    line = next(x for x in open(os.path.join(ROOT, "INTEGRATION.md")).read().splitlines() if x.startswith("last = "))
    got = drafts.Verified(torch.tensor([0, 1, 3, 0, 2], dtype=torch.int32), None,
                          torch.tensor([[-1, -1, -1], [7, -1, -1], [4, 5, 6], [-1, -1, -1], [8, -1, -1]], dtype=torch.int32))
    names = {"torch": torch, "got": got, "last": torch.tensor([11, 12, 13, 14, 15], dtype=torch.int32)}
    exec(line, names)
    assert names["last"].dtype is torch.int32 and names["last"].tolist() == [11, 7, 6, 14, -1]


def test_bad_keeps_are_refused():
    lib = bsa.load()

    def call(heads=2, d=64, path=FAKE, accepted=FAKE, slots=None, rows=4, max_new=8, ws=FAKE, ws_bytes=1 << 30, **kw):
        return lib.bsg_pages_keep(_pool(**kw), heads, d, path, accepted, None, slots, rows, max_new, ws, ws_bytes, None)

    # _pool is of 2 heads of 128
    ok = dict(d=128)
    assert call(rows=0, **ok) == 0
    for bad in (dict(pages=None), dict(scales=None), dict(layers=0), dict(num_pages=0), dict(page_table=None), dict(lengths=None),
                dict(refcounts=None), dict(table_stride=7), dict(path=None), dict(accepted=None), dict(rows=-1), dict(max_new=-1),
                dict(rows=9), dict(page_bytes=4096), dict(page_scales=2), dict(heads=1)):
        assert call(**{**ok, **bad}) in (_lib.BSG_ERR_ARG,), bad
    assert call(d=64) == _lib.BSG_ERR_ARG
    assert call(**ok, pages=FAKE + 4) == _lib.BSG_ERR_ALIGN
    assert call(**ok, page_size=24) == _lib.BSG_ERR_UNSUPPORTED
    assert call(**ok, rows=1025, slots=FAKE) == _lib.BSG_ERR_UNSUPPORTED
    assert call(**ok, max_new=65) == _lib.BSG_ERR_UNSUPPORTED
    over = dict(max_pages=(1 << 26) + 1, table_stride=(1 << 26) + 1)
    assert call(**ok, **over) == _lib.BSG_ERR_UNSUPPORTED
    assert lib.bsg_pages_keep(None, 2, 128, FAKE, FAKE, None, None, 4, 8, FAKE, 1 << 30, None) == _lib.BSG_ERR_ARG
    need = lib.bsg_pages_keep_workspace_bytes(4)
    assert need > 0 and lib.bsg_pages_keep_workspace_bytes(1025) == -1
    assert call(**ok, ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert call(**ok, ws=None) == _lib.BSG_ERR_WORKSPACE
    assert call(**ok, ws=FAKE + 8) == _lib.BSG_ERR_ALIGN


def test_python_layer_refuses_host_tensors():
    x, i = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32)
    pages = torch.zeros(2, 2, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales, tab, n = torch.ones(2, 2, 2), torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    angles = torch.zeros(9, 32)
    with pytest.raises(ValueError):
        bsa.kv_append_rotated(x, x, x, angles, angles, pages, scales, tab, n)
    with pytest.raises(ValueError):
        bsa.kv_tree_attention(x, i, pages, scales, tab, n)
    with pytest.raises(ValueError):
        bsa.verify_drafts(torch.zeros(4, 9), i, torch.zeros(4), max_new=4)
    with pytest.raises(ValueError):
        bsa.pages_keep(pages[None], scales[None], tab, n, n, i.view(4, 1), i)


# ---------------------------------------------------------------------------------------- generated code


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    return {u: _device_asm(u, tmp_path_factory.mktemp("asm")) for u in UNITS}


def test_no_spills_and_no_packed_floats(asm):
    for unit, text in asm.items():
        assert not re.search(r"\bscratch_(load|store)", text), unit
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32", text), unit


def test_tree_steps_wait_for_their_loads(asm):
    """A pair of steps' keys and values come straight into LDS: where waves meet before it, each has waited for all of its
    own, and then asks for the next pair's."""
    found = 0
    for name, body in _functions(asm["kv_tree.hip"], r"_ZN12_GLOBAL__N_118bsg_kv_tree_kernel"):
        d, rows = (int(x) for x in re.findall(r"Li(\d+)E", name))
        pairs = 0
        for i, line in enumerate(body):
            if not line.strip().startswith("s_barrier"):
                continue
            # what comes before the pair's first product, or the next barrier
            after = next((j for j in range(i + 1, len(body)) if "mfma" in body[j] or body[j].strip().startswith("s_barrier")), len(body))
            lines = [j for j in range(i, after) if " lds" in body[j]]
            if after == len(body) or "mfma" not in body[after] or not lines:
                continue
            assert len(lines) == 2 * (2 * d // 64), name
            waited = max(j for j in range(i) if "vmcnt(0)" in body[j])
            assert not any(re.match(r"\s*(buffer|global|flat)_|\.LBB", x) for x in body[waited:i]), name
            pairs += 1
        assert pairs == 2 * rows // 64, (name, pairs)  # large tiles have small ones beside them
        found += 1
    assert found == 8  # two types x two head sizes x two tiles


# ---------------------------------------------------------------------------------------- the oracle


def test_oracle_rotation_is_a_product_of_complex_numbers():
    rng = np.random.default_rng(0)
    x, norm = rng.standard_normal((3, 64)), rng.standard_normal(64)
    angle = rng.standard_normal((10, 16))
    y, _ = dft.turn(x, None, 0.0, np.cos(angle), np.sin(angle), 4, True)
    z = (x[:, 0:32:2] + 1j * x[:, 1:32:2]) * np.exp(1j * angle[4])
    np.testing.assert_allclose(y[:, 0:32:2] + 1j * y[:, 1:32:2], z, rtol=1e-12)
    np.testing.assert_array_equal(y[:, 32:], x[:, 32:])
    y, _ = dft.turn(x, norm, 0.1, np.cos(angle), np.sin(angle), 4, False)
    n = torch.nn.functional.rms_norm(torch.from_numpy(x), (64,), torch.from_numpy(norm), 0.1).numpy()
    z = (n[:, :16] + 1j * n[:, 16:32]) * np.exp(1j * angle[4])
    np.testing.assert_allclose(y[:, :16] + 1j * y[:, 16:32], z, rtol=1e-12)
    np.testing.assert_allclose(y[:, 32:], n[:, 32:], rtol=1e-12)
    assert np.isnan(dft.turn(x, None, 0.0, np.cos(angle), np.sin(angle), 10, False)[0][:, :32]).all()


def test_oracle_chains_are_causal():
    rng = np.random.default_rng(1)
    layer = orc.Layer(rng.integers(0, 100, (4, 2, 2, 16, 64)).astype(np.uint8), np.full((4, 2, 2), 0.125, np.float32))
    q, table, lengths = rng.standard_normal((9, 4, 64)), np.array([[2, 0, 3], [1, -1, -1]]), np.array([40, 9])
    a = orc.attention(q, layer, table, lengths, [0, 5, 9])
    b = dft.tree_attention(q, [-1, 0, 1, 2, 3, -1, 0, 1, 2], layer, table, lengths, [0, 5, 9])
    for x, y in zip(a, b):
        np.testing.assert_allclose(x, y, rtol=1e-13)


def test_oracle_verification_keeps_the_distribution():
    """Over a fine grid of numbers the first token that comes out has the target's probabilities: drafts drawn, and chosen."""
    rng = np.random.default_rng(2)
    p, q = rng.standard_normal((2, 5)), rng.standard_normal((2, 5))
    pp, qq = np.exp(p[0]) / np.exp(p[0]).sum(), np.exp(q[0]) / np.exp(q[0]).sum()
    grid = (np.arange(100) + 0.5) / 100
    share = np.zeros(5)
    for x in range(5):
        for u in grid:
            for v in grid:
                _, _, said = dft.verify(p, [0, x], [v, u], None, q, 1.0, [0, 2])[0]
                share[said[0]] += qq[x] / 1e4
    np.testing.assert_allclose(share, pp, atol=0.02)
    share[:] = 0
    for u in grid[::2]:
        for w in grid[::2]:
            for v in grid[::2]:
                _, _, said = dft.verify(np.concatenate([p, p[:1]]), [0, 3, 1], [v, u, w], [-1, 0, 0], None, 1.0, [0, 3])[0]
                share[said[0]] += 1 / 50 ** 3
    np.testing.assert_allclose(share, pp, atol=0.02)
