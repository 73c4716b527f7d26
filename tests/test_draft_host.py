"""The operators of a step with drafted tokens on the host: their arithmetic under
AddressSanitizer and UndefinedBehaviorSanitizer (tests/sanitize/draft_logic_check.cpp), and
the refusals of their C entries, every one before the device is touched.  Every call starts from one that is right (it gets as far as the missing device)
and changes one thing; the addresses are stand-ins, 1 MiB apart."""
import os
import shutil
import subprocess

import pytest
import torch

import hxm
from hxm import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

INVALID, SHAPE, DTYPE = (_lib.HXM_INVALID_ARG, _lib.HXM_UNSUPPORTED_SHAPE,
                         _lib.HXM_UNSUPPORTED_DTYPE)
REASON = {INVALID: "invalid-argument", SHAPE: "tile-alignment", DTYPE: "unsupported-dtype"}
L = hxm.lib
MB = 1 << 20

pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0,
                                reason="stand-in addresses: only where nothing can launch")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_draft_logic_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "draft_logic_check"
    src = os.path.join(ROOT, "tests", "sanitize", "draft_logic_check.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", src, "-o", str(exe)], check=True, timeout=300)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "draft logic ok" in r.stdout, r.stdout + r.stderr


def _refused(status, want):
    assert status == want, (status, hxm.last_error())
    assert hxm.last_error().startswith(REASON[want])


def pack_heads(h):
    return None if h is None else _lib.HEADS.pack(*h)


def kv(k=24 * MB, v=32 * MB, pages=4, page_size=16, heads=2, dim=64, ks=(2048, 1024, 64),
       vs=(2048, 1024, 64)):
    return _lib.KV_CACHE.pack(k, v, pages, page_size, heads, dim, *ks, *vs)


CACHE = [
    (dict(cache=None), INVALID), (dict(cache=kv(k=0)), INVALID), (dict(cache=kv(v=0)), INVALID),
    (dict(cache=kv(pages=0)), INVALID), (dict(cache=kv(page_size=0)), INVALID),
    (dict(cache=kv(heads=0)), INVALID), (dict(cache=kv(dim=60)), SHAPE),
    (dict(cache=kv(dim=264)), SHAPE), (dict(cache=kv(pages=1 << 27)), SHAPE),
    (dict(cache=kv(heads=65536)), SHAPE), (dict(cache=kv(ks=(2048, 1024, -64))), INVALID),
    (dict(cache=kv(vs=((1 << 40) + 1, 1024, 64))), INVALID), (dict(dtype=hxm.F32), DTYPE),
]
WRITTEN = [
    (dict(cache=kv(ks=(2048, 1024, 63))), INVALID), (dict(cache=kv(vs=(0, 1024, 64))), INVALID),
    (dict(cache=kv(v=24 * MB)), INVALID), (dict(cache=kv(v=24 * MB + 64)), INVALID),
]


def norm_rope(q=(16 * MB, 512, 64), q_out=(17 * MB, 512, 64), q_heads=8, k=(18 * MB, 128, 64),
              v=(19 * MB, 128, 64), q_norm=(1, 1e-6, 20 * MB, 0, 0),
              k_norm=(2, 1e-6, 20 * MB, 21 * MB, 64), positions=22 * MB, cos_sin=23 * MB, ld=64,
              max_pos=100, rot=64, slots=22 * MB, cache=kv(), tokens=5, dtype=hxm.BF16):
    norm = lambda n: None if n is None else _lib.HEAD_NORM.pack(*n)              # noqa: E731
    return L.hxm_norm_rope_append(pack_heads(q), pack_heads(q_out), q_heads, pack_heads(k),
                                  pack_heads(v), norm(q_norm), norm(k_norm), positions, cos_sin, ld,
                                  max_pos, rot, 0, slots, cache, tokens, dtype, None)


@pytest.mark.parametrize("change, status", CACHE + WRITTEN + [
    (dict(tokens=-1), INVALID), (dict(q_heads=-1), INVALID), (dict(tokens=1 << 31), SHAPE),
    (dict(rot=-2), INVALID), (dict(rot=66), INVALID), (dict(rot=63), INVALID),
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=(0, 128, 64)), INVALID),
    (dict(q_out=(17 * MB, 511, 64)), INVALID), (dict(q_out=(18 * MB, 512, 64)), INVALID),
    (dict(q_out=(16 * MB + 2, 512, 64)), INVALID), (dict(max_pos=0), INVALID),
    (dict(ld=63), INVALID), (dict(slots=None), INVALID), (dict(positions=None), INVALID),
    (dict(cos_sin=None), INVALID), (dict(q_norm=None), INVALID), (dict(k_norm=None), INVALID),
    (dict(q_norm=(3, 1e-6, 0, 0, 0)), INVALID), (dict(q_norm=(-1, 1e-6, 0, 0, 0)), INVALID),
    (dict(k_norm=(1, -1e-6, 0, 0, 0)), INVALID), (dict(k_norm=(1, float("nan"), 0, 0, 0)), INVALID),
    (dict(k_norm=(1, 1e-6, 20 * MB, 0, 63)), INVALID),
    (dict(k_norm=(1, 1e-6, 20 * MB, 0, -64)), INVALID),
    (dict(q_norm=(0, 1e-6, 20 * MB, 0, 0)), INVALID), (dict(k_norm=(0, 0.0, 0, 21 * MB, 0)), INVALID),
])
def test_norm_rope_append_refuses(change, status):
    assert norm_rope() == _lib.HXM_NO_DEVICE
    assert norm_rope(q=None, q_out=None, q_heads=0, q_norm=None) == _lib.HXM_NO_DEVICE
    _refused(norm_rope(**change), status)


def tree(q=(16 * MB, 512, 64), out=(17 * MB, 512, 64), q_heads=8, cache=kv(), table=18 * MB, ld=3,
         table_pages=3, lens=19 * MB, parents=20 * MB, batch=2, nodes=5, scale=0.1, window=0,
         lse=21 * MB, dtype=hxm.F16):
    return L.hxm_tree_attention(pack_heads(q), pack_heads(out), q_heads, cache, table, ld,
                                table_pages, lens, parents, batch, nodes, scale, window, lse, dtype,
                                None)


@pytest.mark.parametrize("change, status", CACHE + [
    (dict(batch=-1), INVALID), (dict(nodes=0), INVALID), (dict(nodes=65), SHAPE),
    (dict(q_heads=0), INVALID), (dict(q_heads=7), INVALID), (dict(window=-1), INVALID),
    (dict(batch=1 << 23), SHAPE), (dict(batch=1 << 21, nodes=9), SHAPE), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(q=(0, 512, 64)), INVALID), (dict(q=(16 * MB, -1, 64)), INVALID),
    (dict(out=(17 * MB, 511, 64)), INVALID), (dict(out=(16 * MB, 512, 64)), INVALID),
    (dict(out=(16 * MB + 128, 512, 64)), INVALID), (dict(table_pages=-1), INVALID),
    (dict(ld=2), INVALID), (dict(table=None), INVALID), (dict(lens=None), INVALID),
    (dict(scale=float("nan")), INVALID),
])
def test_tree_attention_refuses(change, status):
    assert tree() == tree(parents=None) == tree(lse=None) == _lib.HXM_NO_DEVICE
    _refused(tree(**change), status)


def verify(tokens=16 * MB, parents=17 * MB, target=18 * MB, ldt=100, draft=19 * MB, ldd=100,
           uniform=20 * MB, path=21 * MB, counts=22 * MB, following=23 * MB, batch=2, nodes=5,
           vocab=100, dtype=hxm.F32):
    return L.hxm_verify_draft(tokens, parents, target, ldt, draft, ldd, uniform, path, counts,
                              following, batch, nodes, vocab, dtype, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=hxm.I8), DTYPE), (dict(batch=-1), INVALID), (dict(nodes=0), INVALID),
    (dict(nodes=65), SHAPE), (dict(vocab=0), INVALID), (dict(vocab=1 << 31, ldt=1 << 31, ldd=1 << 31),
                                                       SHAPE),
    (dict(batch=(1 << 20) + 1), SHAPE), (dict(tokens=None), INVALID), (dict(target=None), INVALID),
    (dict(uniform=None), INVALID), (dict(path=None), INVALID), (dict(counts=None), INVALID),
    (dict(following=None), INVALID), (dict(ldt=99), INVALID), (dict(ldd=99), INVALID),
    (dict(ldt=-100), INVALID),
])
def test_verify_draft_refuses(change, status):
    assert verify() == verify(parents=None, draft=None, ldd=0) == _lib.HXM_NO_DEVICE
    _refused(verify(**change), status)


def compact(cache=kv(), layers=3, kls=8192, vls=8192, table=16 * MB, ld=3, table_pages=3,
            lens=17 * MB, path=18 * MB, counts=19 * MB, lens_out=20 * MB, batch=2, nodes=5,
            dtype=hxm.F16):
    return L.hxm_compact_cache(cache, layers, kls, vls, table, ld, table_pages, lens, path, counts,
                               lens_out, batch, nodes, dtype, None)


LAYERS = [
    (dict(layers=0), INVALID), (dict(layers=65536), INVALID), (dict(kls=8191), INVALID),
    (dict(vls=0), INVALID), (dict(kls=-8192), INVALID), (dict(vls=(1 << 40) + 1), INVALID),
    (dict(cache=kv(v=24 * MB + 2 * 8192 + 2), kls=16384, vls=16384), INVALID),
    (dict(cache=kv(v=24 * MB + 2 * 8192)), INVALID),
]


@pytest.mark.parametrize("change, status", CACHE + WRITTEN + LAYERS + [
    (dict(batch=-1), INVALID), (dict(nodes=0), INVALID), (dict(nodes=65), SHAPE),
    (dict(table_pages=-1), INVALID), (dict(ld=2), INVALID), (dict(table=None), INVALID),
    (dict(lens=None), INVALID), (dict(path=None), INVALID), (dict(counts=None), INVALID),
    (dict(lens_out=17 * MB), INVALID), (dict(lens_out=19 * MB + 4), INVALID),
])
def test_compact_cache_refuses(change, status):
    assert compact() == compact(lens_out=None) == _lib.HXM_NO_DEVICE
    # Keys and values of a layer side by side, of a page, and of a row.
    assert compact(cache=kv(v=24 * MB + 2 * 8192), kls=16384, vls=16384) == _lib.HXM_NO_DEVICE
    assert compact(cache=kv(v=24 * MB + 2 * 2048, ks=(4096, 1024, 64), vs=(4096, 1024, 64)),
                   kls=16384, vls=16384) == _lib.HXM_NO_DEVICE
    assert compact(cache=kv(v=24 * MB + 128, ks=(4096, 2048, 128), vs=(4096, 2048, 128)),
                   kls=16384, vls=16384) == _lib.HXM_NO_DEVICE
    # Layers inside the pages.
    assert compact(cache=kv(ks=(6144, 1024, 64), vs=(6144, 1024, 64)), kls=2048,
                   vls=2048) == _lib.HXM_NO_DEVICE
    _refused(compact(**change), status)


def copy(cache=kv(), layers=3, kls=8192, vls=8192, src=16 * MB, dst=17 * MB, rows=18 * MB, count=4,
         dtype=hxm.F16):
    return L.hxm_copy_pages(cache, layers, kls, vls, src, dst, rows, count, dtype, None)


@pytest.mark.parametrize("change, status", CACHE + WRITTEN + LAYERS + [
    (dict(count=-1), INVALID), (dict(src=None), INVALID), (dict(dst=None), INVALID),
    (dict(count=(1 << 24) + 1), SHAPE),
    (dict(cache=kv(v=1 << 40, pages=1, page_size=1 << 30, heads=1, dim=64), layers=1), SHAPE),
])
def test_copy_pages_refuses(change, status):
    assert copy() == copy(rows=None) == _lib.HXM_NO_DEVICE
    _refused(copy(**change), status)
