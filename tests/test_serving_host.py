"""The serving operators' C ABI and oracle without a GPU: the header and its ctypes mirror agree, calls
that cannot be right are refused on the host, and oracle/serving.py matches independent forms."""
from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess
import threading

import numpy as np
import pytest
import torch

import bsa_mi355x as bsa
from bsa_mi355x import _lib, serving
from oracle import serving as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "bsgserve.h")
FAKE = 1 << 40  # never dereferenced: every call below fails validation first


def test_header_and_library_agree(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(bsg_[a-z0-9_]+)\s*\(", text))
    assert len(names) == 11
    lib = bsa.load()
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES, name
    assert serving.COUNTER_BYTES == int(re.search(r"BSG_KV_COUNTER_BYTES (\d+)", text).group(1))
    assert serving.MAX_ROWS == int(re.search(r"BSG_PAGES_MAX_ROWS (\d+)", text).group(1))
    assert serving.MAX_ALTERNATIVES == int(re.search(r"BSG_LOGPROBS_MAX_K (\d+)", text).group(1))
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("gcc not available")
    src, exe = tmp_path / "s.c", tmp_path / "s"
    fields = {"bsg_kv_cache": _lib.KvCache, "bsg_page_pool": _lib.PagePool}
    prints = "".join(f'printf("%zu\\n", sizeof({t}));' + "".join(f'printf("%zu\\n", offsetof({t}, {f}));' for f, _ in c._fields_)
                     for t, c in fields.items())
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "bsgserve.h"\nint main(void){' + prints + "return 0;}")
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()))
    want = []
    for c in fields.values():
        want += [ctypes.sizeof(c)] + [getattr(c, f).offset for f, _ in c._fields_]
    assert got == want


def _cache(**kw):
    a = dict(pages=FAKE, scales=FAKE, num_pages=10, n_heads=2, page_size=16, head_dim=128, num_slots=4, max_pages=8,
             table_stride=8, page_table=FAKE, lengths=FAKE)
    a.update(kw)
    return _lib.KvCache(*a.values())


BAD_CACHES = [(dict(pages=None), _lib.BSG_ERR_ARG), (dict(lengths=None), _lib.BSG_ERR_ARG), (dict(num_pages=0), _lib.BSG_ERR_ARG),
              (dict(table_stride=7), _lib.BSG_ERR_ARG), (dict(page_size=24), _lib.BSG_ERR_UNSUPPORTED),
              (dict(head_dim=96), _lib.BSG_ERR_UNSUPPORTED), (dict(pages=FAKE + 8), _lib.BSG_ERR_ALIGN),
              (dict(scales=FAKE + 4), _lib.BSG_ERR_ALIGN), (dict(max_pages=1 << 28, table_stride=1 << 28), _lib.BSG_ERR_UNSUPPORTED)]


def _append(cache, k=FAKE, tokens=4, rows=4, cu=None, max_new=1, dtype=0, slots=None):
    return bsa.load().bsg_kv_append(k, 256, 128, FAKE, 256, 128, tokens, ctypes.byref(cache), slots, rows, cu, max_new, dtype, None)


def _attend(cache, q=FAKE, qs=(512, 128), tokens=4, heads=4, rows=4, cu=None, max_new=1, out=FAKE, os_=(512, 128), dtype=0,
            ws=FAKE, ws_bytes=1 << 40, cus=256, slots=None, max_len=0):
    return bsa.load().bsg_kv_attention(q, *qs, tokens, heads, ctypes.byref(cache), slots, rows, cu, max_new, max_len, 0.1, out, *os_,
                                       None, dtype, ws, ws_bytes, cus, None)


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_bad_caches_are_refused(bad, code):
    assert _append(_cache(**bad)) == code
    assert _attend(_cache(**bad)) == code
    assert bsa.load().bsg_kv_attention_workspace_bytes(ctypes.byref(_cache(**bad)), 4, 4, 1, 0, 256) == -1
    assert _lib.last_error()


def test_rows_of_more_than_2_30_tokens_are_refused():
    """Positions are 32-bit in the attention, and go past a row's end by up to a few thousand."""
    over, most = (_cache(max_pages=n, table_stride=n) for n in ((1 << 26) + 1, 1 << 26))
    assert _append(over) == _lib.BSG_ERR_UNSUPPORTED and _attend(over) == _lib.BSG_ERR_UNSUPPORTED
    need = bsa.load().bsg_kv_attention_workspace_bytes
    assert need(ctypes.byref(over), 4, 4, 1, 0, 256) == -1 and need(ctypes.byref(most), 4, 4, 1, 0, 256) > 0


def test_page_calls_refuse_the_rows_that_append_and_attention_refuse():
    lib = bsa.load()
    over, most = (dict(max_pages=n, table_stride=n) for n in ((1 << 26) + 1, 1 << 26))
    need = lib.bsg_pages_workspace_bytes(100)
    for sizes, code in ((over, _lib.BSG_ERR_UNSUPPORTED), (most, _lib.BSG_ERR_WORKSPACE)):
        assert lib.bsg_pages_extend(_pool(**sizes), FAKE, FAKE, 4, FAKE, FAKE, need - 1, None) == code
        assert lib.bsg_pages_compact(_pool(**sizes), FAKE, FAKE, need - 1, None) == code
    assert lib.bsg_pages_fork(_pool(**over), FAKE, FAKE, 4, None) == _lib.BSG_ERR_UNSUPPORTED
    assert lib.bsg_pages_free(_pool(**over), FAKE, 4, None) == _lib.BSG_ERR_UNSUPPORTED


def test_bad_batches_are_refused():
    c = _cache()
    assert _append(c, k=None) == _lib.BSG_ERR_ARG
    assert _append(c, dtype=2) == _lib.BSG_ERR_DTYPE
    assert _append(c, tokens=5) == _lib.BSG_ERR_ARG
    assert _append(c, rows=5, tokens=5) == _lib.BSG_ERR_ARG  # more rows than slots
    assert _append(c, max_new=-1, cu=FAKE) == _lib.BSG_ERR_ARG
    assert _append(c, k=FAKE + 1) == _lib.BSG_ERR_ALIGN
    assert _append(c, tokens=0, rows=0) == 0
    assert _attend(c, heads=3) == _lib.BSG_ERR_ARG
    assert _attend(c, heads=0) == _lib.BSG_ERR_ARG
    assert _attend(c, q=None) == _lib.BSG_ERR_ARG
    assert _attend(c, cus=0) == _lib.BSG_ERR_ARG
    assert _attend(c, q=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert _attend(c, qs=(512, 132)) == _lib.BSG_ERR_ALIGN
    assert _attend(c, out=FAKE + 4) == _lib.BSG_ERR_ALIGN
    assert _attend(c, os_=(514, 128)) == _lib.BSG_ERR_ALIGN
    assert _attend(c, dtype=7) == _lib.BSG_ERR_DTYPE
    assert _attend(c, rows=70000, tokens=70000, slots=FAKE) == _lib.BSG_ERR_UNSUPPORTED
    assert _attend(c, max_new=0, tokens=0) == 0
    long = _cache(max_pages=4096, table_stride=4096)
    need = bsa.load().bsg_kv_attention_workspace_bytes(ctypes.byref(long), 4, 4, 1, 0, 256)
    assert need > serving.COUNTER_BYTES
    assert _attend(long, ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert _attend(long, ws=None) == _lib.BSG_ERR_WORKSPACE
    assert _attend(long, ws=FAKE + 8) == _lib.BSG_ERR_ALIGN


def _pool(**kw):
    a = dict(pages=FAKE, scales=FAKE, layers=2, num_pages=100, page_bytes=8192, page_scales=4, page_size=16, num_slots=8, max_pages=8,
             table_stride=8, page_table=FAKE, lengths=FAKE, refcounts=FAKE)
    a.update(kw)
    return ctypes.byref(_lib.PagePool(*a.values()))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_refuses_a_scale_that_is_no_number(scale, new):
    """The prompt kernel would read NaN as 0."""
    rc = bsa.load().bsg_kv_attention(FAKE, 512, 128, 4 * new, 4, ctypes.byref(_cache()), None, 4, None, new, 0, scale, FAKE, 512, 128,
                                     None, 0, FAKE, 1 << 40, 256, None)
    assert rc == _lib.BSG_ERR_ARG and "sm_scale" in _lib.last_error()


def test_launches_of_too_many_threads_are_refused():
    """The machine cuts a launch of 2^32 threads short without an error."""
    wide = _cache(n_heads=4096)
    assert _attend(wide, heads=4096, rows=1, tokens=1 << 19, max_new=1 << 19) == _lib.BSG_ERR_UNSUPPORTED
    flat = _pool(page_size=1, max_pages=1 << 28, table_stride=1 << 28)
    assert bsa.load().bsg_pages_fork(flat, FAKE, FAKE, 4, None) == _lib.BSG_ERR_UNSUPPORTED


def test_append_of_too_much_work_is_refused():
    """A bound on the new tokens near 2^31 is counted in 64 bits."""
    for most in (2 ** 31 - 1, 2 ** 31 - 14):
        assert _append(_cache(), cu=FAKE, max_new=most) == _lib.BSG_ERR_UNSUPPORTED


def test_bad_pools_are_refused():
    lib = bsa.load()
    need = lib.bsg_pages_workspace_bytes(100)
    assert need > 0 and lib.bsg_pages_workspace_bytes(0) == -1 and lib.bsg_pages_workspace_bytes(1 << 31) == -1

    def extend(p, n=4, slots=FAKE, new=FAKE, served=FAKE, ws=FAKE, ws_bytes=need):
        return lib.bsg_pages_extend(p, slots, new, n, served, ws, ws_bytes, None)

    for bad in (dict(pages=None), dict(scales=None), dict(layers=0), dict(page_bytes=24), dict(num_pages=0), dict(page_table=None),
                dict(lengths=None), dict(refcounts=None), dict(table_stride=7), dict(page_size=0)):
        assert extend(_pool(**bad)) == _lib.BSG_ERR_ARG, bad
    assert extend(_pool(pages=FAKE + 4)) == _lib.BSG_ERR_ALIGN
    assert extend(_pool(), n=1025) == _lib.BSG_ERR_UNSUPPORTED
    assert extend(_pool(), n=-1) == _lib.BSG_ERR_ARG
    assert extend(_pool(), n=9, slots=None) == _lib.BSG_ERR_ARG
    assert extend(_pool(), new=None) == _lib.BSG_ERR_ARG
    assert extend(_pool(), ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert extend(_pool(), ws=FAKE + 8) == _lib.BSG_ERR_ALIGN
    assert lib.bsg_pages_compact(_pool(), None, FAKE, need, None) == _lib.BSG_ERR_ARG
    assert lib.bsg_pages_compact(_pool(), FAKE, None, need, None) == _lib.BSG_ERR_WORKSPACE
    assert lib.bsg_pages_fork(_pool(), FAKE, FAKE, 1025, None) == _lib.BSG_ERR_UNSUPPORTED
    assert lib.bsg_pages_fork(_pool(), None, FAKE, 2, None) == _lib.BSG_ERR_ARG
    assert lib.bsg_pages_free(_pool(), None, 2, None) == _lib.BSG_ERR_ARG
    assert lib.bsg_pages_copy(_pool(), FAKE, None, 2, None) == _lib.BSG_ERR_ARG
    assert lib.bsg_pages_copy(_pool(), FAKE, FAKE, -2, None) == _lib.BSG_ERR_ARG
    assert lib.bsg_pages_copy(None, FAKE, FAKE, 2, None) == _lib.BSG_ERR_ARG


def test_bad_logprobs_are_refused():
    lib = bsa.load()

    def call(x=FAKE, rows=4, vocab=1 << 20, k=3, ids=FAKE, dtype=0, ws=FAKE, ws_bytes=1 << 30, cus=256):
        return lib.bsg_token_logprobs(x, vocab, rows, vocab, FAKE, k, FAKE, FAKE, ids, FAKE, dtype, ws, ws_bytes, cus, None)

    assert call(x=None) == _lib.BSG_ERR_ARG
    assert call(ids=None) == _lib.BSG_ERR_ARG
    assert call(k=65) == _lib.BSG_ERR_UNSUPPORTED
    assert call(vocab=2) == _lib.BSG_ERR_ARG  # k > vocab
    assert call(rows=-1) == _lib.BSG_ERR_ARG
    assert call(dtype=3) == _lib.BSG_ERR_DTYPE
    assert call(cus=0) == _lib.BSG_ERR_ARG
    assert call(x=FAKE + 1) == _lib.BSG_ERR_ALIGN
    assert call(x=FAKE + 2, dtype=2) == _lib.BSG_ERR_ALIGN
    assert call(ws=None) == _lib.BSG_ERR_WORKSPACE
    need = lib.bsg_token_logprobs_workspace_bytes(4, 1 << 20, 3, 0, 256)
    assert need > 0 and call(ws_bytes=need - 1) == _lib.BSG_ERR_WORKSPACE
    assert call(rows=0) == 0
    assert lib.bsg_token_logprobs_workspace_bytes(0, 1 << 20, 3, 0, 256) == 0


def test_python_layer_refuses_host_tensors():
    with pytest.raises(ValueError):
        bsa.token_logprobs(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int32))
    pages = torch.zeros(2, 1, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    tab, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        bsa.kv_attention(torch.zeros(1, 1, 64, dtype=torch.float16), pages, torch.ones(2, 1, 2), tab, n)
    with pytest.raises(ValueError):
        bsa.pages_free(tab, n, n, n)


class _Device:
    """torch's current device, streams and capture as a test sets them; workspaces are host tensors."""

    def __init__(self, monkeypatch):
        self.current, self.capturing = 0, set()
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 * index, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: self.current in self.capturing, raising=False)
        for name in ("zeros", "empty"):
            def make(*a, real=getattr(torch, name), device=None, **kw):
                return real(*a, **kw)
            monkeypatch.setattr(serving.torch, name, make)
        outer = self

        class Guard:
            def __init__(self, index):
                self.index = index

            def __enter__(self):
                self.was, outer.current = outer.current, self.index

            def __exit__(self, *_):
                outer.current = self.was

        monkeypatch.setattr(torch.cuda, "device", Guard)


def test_threads_on_one_stream_have_workspaces_of_their_own(monkeypatch):
    """extend and compact hand a plan from one launch to the next in the workspace: what another thread
    enqueues on the same stream in between must not write there."""
    _Device(monkeypatch)
    mine = serving._workspace(0, 5000, None)
    assert serving._workspace(0, 5000, None) is mine
    theirs = []
    threads = [threading.Thread(target=lambda: theirs.append(serving._workspace(0, 5000, None))) for _ in range(2)]
    for t in threads:
        t.start()
        t.join()
    assert len({t.data_ptr() for t in (mine, *theirs)}) == 3


def test_workspace_asks_the_tensors_device_for_a_capture(monkeypatch):
    """Not the current one: a call on device 1 from device 0."""
    d = _Device(monkeypatch)
    eager = serving._workspace(1, 5000, None)
    d.capturing = {1}
    first, second = (serving._workspace(1, 5000, None) for _ in range(2))
    assert first is not eager and second is not first and first.numel() == 5000
    assert serving._workspace(0, 5000, None) is serving._workspace(0, 5000, None)
    d.capturing = {0}
    assert serving._workspace(1, 5000, None) is eager
    with pytest.raises(RuntimeError):
        serving._workspace(0, 5000, "not used before")
    assert serving._workspace(1, 5000, "not used before") is not None and d.current == 0


def test_oracle_e4m3_is_torchs():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(orc.E4M3, table)
    x = np.concatenate([np.random.default_rng(0).standard_normal(20000) * np.exp(np.linspace(-8, 4, 20000)),
                        (orc.E4M3[:126] + orc.E4M3[1:127]) / 2, [0.0, -0.0, 448, 464, 1e9, -1e9, np.inf, -np.inf, np.nan]])
    want = torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(orc.round_e4m3(x.astype(np.float32)), want)
    for a in (1e-30, 0.3, 447.9, 448.0, 448.1, 7.0, 1e38):
        s = orc.scale_for(a)
        assert s == 2.0 ** -40 or s == 2.0 ** 80 or (a <= 448 * s and a > 224 * s)


def test_oracle_layout_is_what_read_pages_undoes():
    rng = np.random.default_rng(1)
    raw = rng.integers(0, 120, (3, 2, 2, 32, 128)).astype(np.uint8)
    scales = 2.0 ** rng.integers(-3, 3, (3, 2, 2)).astype(np.float32)
    layer = orc.Layer(raw, scales)
    np.testing.assert_array_equal(layer.tiled(), orc.E4M3[raw])
    k, v = bsa.read_pages(torch.from_numpy(raw).view(torch.float8_e4m3fn), torch.from_numpy(scales))
    for i, x in enumerate((k, v)):
        np.testing.assert_array_equal(x.double().numpy(), layer.values[:, :, i] * layer.scales[:, :, i][..., None, None])


def test_oracle_attention_and_logprobs_match_torch():
    rng = np.random.default_rng(2)
    raw = rng.integers(0, 100, (4, 1, 2, 16, 64)).astype(np.uint8)
    layer = orc.Layer(raw, np.full((4, 1, 2), 0.125, np.float32))
    q = rng.standard_normal((5, 2, 64))
    out, lse, *_ = orc.attention(q, layer, np.array([[2, 0, 3]]), np.array([40]), [0, 5])
    k, v = (torch.from_numpy(layer.values[[2, 0, 3], 0, i].reshape(48, 64)[:40] * 0.125) for i in (0, 1))
    x = torch.from_numpy(q).permute(1, 0, 2) @ k.t() / 8
    x.masked_fill_(torch.arange(40)[None] > torch.arange(35, 40)[:, None], float("-inf"))
    np.testing.assert_allclose(out, (x.softmax(-1) @ v).permute(1, 0, 2).numpy(), rtol=1e-12, atol=1e-14)
    np.testing.assert_allclose(lse, x.logsumexp(-1).t().numpy(), rtol=1e-12)
    logits = rng.standard_normal((6, 50))
    lp, ent, ids, top = orc.token_logprobs(logits, np.arange(6), 5)
    d = torch.distributions.Categorical(logits=torch.from_numpy(logits))
    np.testing.assert_allclose(lp, d.log_prob(torch.arange(6)).numpy(), rtol=1e-12)
    np.testing.assert_allclose(ent, d.entropy().numpy(), rtol=1e-12)
    t = torch.from_numpy(logits).log_softmax(-1).topk(5)
    np.testing.assert_array_equal(ids, t.indices.numpy())
    np.testing.assert_allclose(top, t.values.numpy(), rtol=1e-12)


def test_oracle_pool_keeps_its_counts():
    """After any steps the counts are those of the table, and no page written next has two readers."""
    rng = np.random.default_rng(3)
    pool = orc.Pool([[-1] * 6] * 9, [0] * 9, [0] * 30, 4, range(30))
    for _ in range(200):
        kind = rng.integers(4)
        if kind == 0:
            pool.fork(rng.integers(-1, 10, 3).tolist(), rng.integers(-1, 10, 3).tolist())
        elif kind == 1:
            slots = rng.permutation(9)[:4].tolist()
            new = rng.integers(0, 7, 4).tolist()
            for s, ok, n in zip(slots, pool.extend(new, slots), new):
                if ok and n:
                    first = (pool.lengths[s] - n) // 4
                    assert all(pool.refs[pool.table[s][j]] == 1 for j in range(first, -(-pool.lengths[s] // 4)))
        elif kind == 2:
            pool.free(rng.integers(-1, 10, 2).tolist())
        else:
            live, _ = pool.compact()
            assert all(r > 0 for r in pool.refs[:live]) and not any(pool.refs[live:])
        named = [x for r in pool.table for x in r if x >= 0]
        assert pool.refs == [named.count(i) for i in range(30)]
