"""The decoder-layer operators on the host: their arithmetic under
AddressSanitizer and UndefinedBehaviorSanitizer
(tests/sanitize/decoder_logic_check.cpp: overlap rules, division by
multiplication, paged attention's cut of a batch), and the refusals of their C
entries, every one before the device is touched."""
import os
import shutil
import subprocess

import pytest
import torch

import hxm
import hxm.ops
from hxm import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, SHAPE, DTYPE = (_lib.HXM_INVALID_ARG, _lib.HXM_UNSUPPORTED_SHAPE,
                         _lib.HXM_UNSUPPORTED_DTYPE)
REASON = {INVALID: "invalid-argument", SHAPE: "tile-alignment", DTYPE: "unsupported-dtype"}
L = hxm.lib
MB = 1 << 20


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_decoder_logic_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "decoder_logic_check"
    src = os.path.join(ROOT, "tests", "sanitize", "decoder_logic_check.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", src, "-o", str(exe)], check=True, timeout=300)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "decoder logic ok" in r.stdout, r.stdout + r.stderr


def _refused(status, want, words=""):
    assert status == want, (status, hxm.last_error())
    assert hxm.last_error().startswith(REASON[want]) and words in hxm.last_error()


no_gpu = pytest.mark.skipif(torch.cuda.device_count() > 0,
                            reason="stand-in addresses: only where nothing can launch")


# Every call below starts from one that is right (it gets as far as the missing
# device) and changes one thing.  The addresses are stand-ins, 1 MiB apart.

def residual(h=16 * MB, ldh=64, x=17 * MB, ldx=64, post=(1, 1e-6, 18 * MB, 0), gate=19 * MB, ldg=64,
             gate_rows=1, pre=(2, 1e-6, 20 * MB, 21 * MB), y=22 * MB, ldy=64, z=23 * MB, ldz=64,
             rows=8, cols=64, dtype=hxm.F16):
    norm = lambda n: None if n is None else _lib.ROW_NORM.pack(*n)  # noqa: E731
    return L.hxm_residual_norm_rows(h, ldh, x, ldx, norm(post), gate, ldg, gate_rows, 1.0, 1.0,
                                    norm(pre), y, ldy, z, ldz, rows, cols, dtype, None)


RESIDUAL = [
    (dict(dtype=hxm.I8), DTYPE), (dict(post=None), INVALID), (dict(pre=None), INVALID),
    (dict(post=(3, 1e-6, 0, 0)), INVALID), (dict(pre=(-1, 1e-6, 0, 0)), INVALID),
    (dict(post=(0, 1e-6, 18 * MB, 0)), INVALID), (dict(pre=(1, -1e-6, 0, 0)), INVALID),
    (dict(pre=(1, float("nan"), 0, 0)), INVALID),
    (dict(rows=-1), INVALID), (dict(cols=0), INVALID), (dict(gate_rows=-1), INVALID),
    (dict(rows=1 << 31), SHAPE), (dict(h=None), INVALID), (dict(x=None), INVALID),
    (dict(y=None), INVALID), (dict(z=None), INVALID), (dict(gate=None), INVALID),
    (dict(gate_rows=0), INVALID), (dict(pre=(0, 0.0, 0, 0)), INVALID),
    (dict(ldh=63), INVALID), (dict(ldx=63), INVALID), (dict(ldy=63), INVALID),
    (dict(ldz=63), INVALID), (dict(ldg=63), INVALID), (dict(ldh=(1 << 40) + 1), INVALID),
    (dict(gate_rows=3), INVALID),
    (dict(y=16 * MB + 2), INVALID), (dict(z=17 * MB - 2), INVALID),
    (dict(y=23 * MB + 128), INVALID),
    (dict(y=16 * MB, ldy=65), INVALID), (dict(y=23 * MB), INVALID),
]


@no_gpu
@pytest.mark.parametrize("change, status", RESIDUAL)
def test_residual_norm_refuses(change, status):
    _refused(residual(**change), status)


def rope(q=(16 * MB, 512, 64), q_out=(17 * MB, 512, 64), q_heads=8, k=(18 * MB, 128, 64),
         v=(19 * MB, 128, 64), positions=20 * MB, cos_sin=21 * MB, ld=64, max_pos=100, rot=64,
         slots=22 * MB, k_cache=24 * MB, v_cache=25 * MB, pages=4, page_size=16, heads=2, dim=64,
         ks=(2048, 1024, 64), vs=(2048, 1024, 64), tokens=5, dtype=hxm.BF16, cache=True):
    pack = lambda h: None if h is None else _lib.HEADS.pack(*h)  # noqa: E731
    c = _lib.KV_CACHE.pack(k_cache, v_cache, pages, page_size, heads, dim, *ks, *vs)
    return L.hxm_rope_append(pack(q), pack(q_out), q_heads, pack(k), pack(v), positions, cos_sin, ld,
                             max_pos, rot, 0, slots, c if cache else None, tokens, dtype, None)


CACHE = [
    (dict(cache=False), INVALID), (dict(k_cache=0), INVALID), (dict(v_cache=0), INVALID),
    (dict(pages=0), INVALID), (dict(page_size=0), INVALID), (dict(heads=0), INVALID),
    (dict(dim=0), INVALID), (dict(dim=60), SHAPE), (dict(dim=264), SHAPE),
    (dict(pages=1 << 27), SHAPE), (dict(pages=1 << 40, page_size=1 << 40), SHAPE),
    (dict(heads=65536), SHAPE), (dict(ks=(2048, 1024, -64)), INVALID),
    (dict(vs=((1 << 40) + 1, 1024, 64)), INVALID),
]
ROPE = CACHE + [
    (dict(dtype=hxm.F32), DTYPE),
    (dict(ks=(2048, 1024, 63)), INVALID), (dict(vs=(0, 1024, 64)), INVALID),
    (dict(ks=(2048, 64, 64)), INVALID),
    (dict(tokens=-1), INVALID), (dict(q_heads=-1), INVALID), (dict(tokens=1 << 31), SHAPE),
    (dict(q_heads=65536), SHAPE), (dict(rot=-2), INVALID), (dict(rot=66), INVALID),
    (dict(rot=63), INVALID), (dict(q=None), INVALID), (dict(q_out=None), INVALID),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(q=(0, 512, 64)), INVALID),
    (dict(k=(18 * MB, -1, 64)), INVALID), (dict(q_out=(17 * MB, 511, 64)), INVALID),
    (dict(q_out=(17 * MB, 512, 63)), INVALID), (dict(max_pos=0), INVALID), (dict(ld=63), INVALID),
    (dict(positions=None), INVALID), (dict(cos_sin=None), INVALID), (dict(slots=None), INVALID),
    (dict(q_out=(16 * MB + 16, 512, 64)), INVALID), (dict(q_out=(16 * MB, 576, 64)), INVALID),
    (dict(q_out=(18 * MB - 64, 512, 64)), INVALID), (dict(q_out=(19 * MB, 512, 64)), INVALID),
]


@no_gpu
@pytest.mark.parametrize("change, status", ROPE)
def test_rope_append_refuses(change, status):
    _refused(rope(**change), status)


def attention(q=(16 * MB, 512, 64), out=(17 * MB, 512, 64), q_heads=8, k_cache=24 * MB,
              v_cache=25 * MB, pages=4, page_size=16, heads=2, dim=64, ks=(2048, 1024, 64),
              vs=(2048, 1024, 64), table=18 * MB, ld=3, table_pages=3, lens=19 * MB, batch=5,
              scale=0.125, window=0, dtype=hxm.F16, cache=True):
    pack = lambda h: None if h is None else _lib.HEADS.pack(*h)  # noqa: E731
    c = _lib.KV_CACHE.pack(k_cache, v_cache, pages, page_size, heads, dim, *ks, *vs)
    return L.hxm_paged_attention(pack(q), pack(out), q_heads, c if cache else None, table, ld,
                                 table_pages, lens, batch, scale, window, None, dtype, None)


ATTENTION = CACHE + [
    (dict(dtype=hxm.F32), DTYPE), (dict(batch=-1), INVALID), (dict(q_heads=0), INVALID),
    (dict(q_heads=7), INVALID), (dict(window=-1), INVALID), (dict(q_heads=65538), SHAPE),
    (dict(batch=(1 << 24) + 1), SHAPE), (dict(batch=1 << 22), SHAPE), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(q=(0, 512, 64)), INVALID), (dict(out=(0, 512, 64)), INVALID),
    (dict(out=(17 * MB, 511, 64)), INVALID), (dict(out=(16 * MB, 520, 64)), INVALID),
    (dict(out=(16 * MB + 2, 512, 64)), INVALID), (dict(table=None), INVALID),
    (dict(lens=None), INVALID), (dict(table_pages=-1), INVALID), (dict(table_pages=1 << 31), INVALID),
    (dict(ld=2), INVALID), (dict(ld=-1), INVALID), (dict(scale=float("nan")), INVALID),
]


@no_gpu
@pytest.mark.parametrize("change, status", ATTENTION)
def test_paged_attention_refuses(change, status):
    _refused(attention(**change), status)


def lora(y=16 * MB, ldy=48, x=17 * MB, ldx=64, A=18 * MB, B=19 * MB, adapters=3, R=16, index=20 * MB,
         scale=21 * MB, out=22 * MB, ldo=48, M=9, N=48, K=64, dtype=hxm.F16):
    return L.hxm_lora_add(y, ldy, x, ldx, A, B, adapters, R, index, scale, out, ldo, M, N, K, dtype,
                          None)


LORA = [
    (dict(dtype=hxm.F32), DTYPE), (dict(M=-1), INVALID), (dict(N=-1), INVALID), (dict(K=0), INVALID),
    (dict(adapters=-1), INVALID), (dict(R=0), INVALID), (dict(R=12), SHAPE), (dict(R=264), SHAPE),
    (dict(K=60), SHAPE), (dict(M=1 << 30), SHAPE), (dict(N=1 << 30), SHAPE), (dict(K=1 << 30), SHAPE),
    (dict(adapters=1 << 30), SHAPE), (dict(ldy=47), INVALID), (dict(ldx=63), INVALID),
    (dict(ldo=47), INVALID), (dict(ldx=(1 << 40) + 1), INVALID), (dict(y=None), INVALID),
    (dict(x=None), INVALID), (dict(A=None), INVALID), (dict(B=None), INVALID),
    (dict(index=None), INVALID), (dict(out=None), INVALID), (dict(out=16 * MB, ldo=49), INVALID),
    (dict(out=16 * MB + 2), INVALID), (dict(out=17 * MB), INVALID), (dict(out=17 * MB + 1024), INVALID),
]


@no_gpu
@pytest.mark.parametrize("change, status", LORA)
def test_lora_add_refuses(change, status):
    _refused(lora(**change), status)


@no_gpu
def test_right_calls_get_as_far_as_the_device():
    calls = [
        residual(), residual(y=16 * MB, z=17 * MB), residual(rows=0, h=None, x=None, y=None),
        residual(gate=None, gate_rows=0), residual(gate_rows=8), residual(gate_rows=4),
        residual(pre=(0, 0.0, 0, 0), z=None), residual(cols=1, rows=1, y=16 * MB, ldy=99),
        residual(h=16 * MB, ldh=128, y=16 * MB + 128, ldy=128),  # columns side by side
        rope(), rope(q=(16 * MB, 512, 64), q_out=(16 * MB, 512, 64)), rope(q=None, q_out=None, q_heads=0),
        rope(rot=0, positions=None, cos_sin=None), rope(tokens=0, slots=None),
        rope(ks=(2048, 64, 128), vs=(1024, 4096, 64)),
        rope(k=(18 * MB, 0, 0), v=(18 * MB, 0, 0)),  # broadcast inputs
        attention(), attention(out=(16 * MB, 512, 64)), attention(ld=0, batch=1),
        attention(table=None, table_pages=0, ld=0), attention(window=1 << 40),
        attention(k_cache=24 * MB, v_cache=24 * MB), attention(batch=0, lens=None, table=None),
        lora(), lora(out=16 * MB), lora(M=0, y=None), lora(N=0, ldy=0, ldo=0, x=None),
        lora(adapters=0, A=None, B=None), lora(scale=None),
    ]
    assert all(c == _lib.HXM_NO_DEVICE for c in calls), calls


def test_host_tensors_are_refused():
    t = torch.zeros(4, 2, 64, dtype=torch.float16)
    cache = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: hxm.ops.residual_norm(t, t),
                 lambda: hxm.ops.rope_append(t, t, t, cache, cache, i),
                 lambda: hxm.ops.paged_attention(t, cache, cache, i.view(4, 1), i),
                 lambda: hxm.ops.lora_add(t[:, 0], t[:, 0], t, t, i)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def interleaved(heads, tokens=5, **kw):
    """A fused projection whose heads hold q, k and v side by side ([tokens, heads, 3, 64]),
    q turned in place."""
    at = lambda i: (16 * MB + 128 * i, heads * 192, 192)  # noqa: E731
    return rope(**{**dict(q=at(0), q_out=at(0), q_heads=heads, k=at(1), v=at(2), heads=heads,
                          ks=(heads * 1024, 1024, 64), vs=(heads * 1024, 1024, 64),
                          tokens=tokens), **kw})


@no_gpu
@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("heads", [1, 2, 8])
def test_rope_append_in_place_between_the_heads_of_k_and_v(heads, tokens):
    assert interleaved(heads, tokens) == _lib.HXM_NO_DEVICE, hxm.last_error()
    # k a dim short of q's end, and (where there is a next head) past its start.
    for off in (63, 129):
        st = interleaved(heads, tokens, k=(16 * MB + 2 * off, heads * 192, 192),
                         v=(19 * MB, heads * 192, 192))
        if off == 63 or heads * tokens > 1:
            _refused(st, INVALID, "overlaps")
        else:
            assert st == _lib.HXM_NO_DEVICE


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_overlap_logic_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "overlap_logic_check"
    src = os.path.join(ROOT, "tests", "sanitize", "overlap_logic_check.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", src, "-o", str(exe)], check=True, timeout=300)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "overlap logic ok" in r.stdout, r.stdout + r.stderr


KV = dict(pages=4, page_size=16, heads=2, dim=64)


@no_gpu
@pytest.mark.parametrize("v_cache, ks, vs", [
    (24 * MB, (2048, 1024, 64), (2048, 1024, 64)),               # one cache for both
    (24 * MB, (2048, 1024, 64), (2048, 64, 128)),                # in two layouts
    (24 * MB + 2, (2048, 1024, 64), (2048, 1024, 64)),
    (24 * MB + 2 * 1024, (2048, 1024, 64), (2048, 1024, 64)),    # values at the next head's keys
    (24 * MB + 2 * 2048, (2048, 1024, 64), (2048, 1024, 64)),    # at the next page's
    (24 * MB - 2 * 2048, (2048, 1024, 64), (2048, 1024, 64)),
    (24 * MB + 2 * 2040, (4096, 1024, 64), (4096, 1024, 64)),    # eight elements into the page
])
def test_rope_append_refuses_keys_and_values_in_one_place(v_cache, ks, vs):
    _refused(rope(**KV, v_cache=v_cache, ks=ks, vs=vs), INVALID, "keys and values")
    # Attention only reads them.
    assert attention(**KV, v_cache=v_cache, ks=ks, vs=vs) == _lib.HXM_NO_DEVICE


@no_gpu
@pytest.mark.parametrize("at, ks, vs", [
    (8192, (2048, 1024, 64), (2048, 1024, 64)),                  # [2, pages, heads, page, dim]
    (-8192, (2048, 1024, 64), (2048, 1024, 64)),
    (2048, (4096, 1024, 64), (4096, 1024, 64)),                  # [pages, 2, heads, page, dim]
    (-2048, (4096, 64, 128), (4096, 64, 128)),                   # [pages, 2, page, heads, dim]
    (2048, (4096, 1024, 64), (4096, 64, 128)),                   # each half in its own layout
    (1024, (4096, 2048, 64), (4096, 2048, 64)),                  # [pages, heads, 2, page, dim]
    (64, (4096, 2048, 128), (4096, 2048, 128)),                  # [pages, heads, page, 2, dim]
    (64, (4096, 128, 256), (4096, 128, 256)),                    # [pages, page, heads, 2, dim]
    (128, (4096, 64, 256), (4096, 64, 256)),                     # [pages, page, 2, heads, dim]
    (3 * 2048, (4 * 2048, 1024, 64), (4 * 2048, 1024, 64)),      # of [pages, layers, 2, ..]
    (3 * 2048, (4096, 1024, 64), (4096, 1024, 64)),              # values a page further
])
def test_rope_append_takes_keys_and_values_side_by_side(at, ks, vs):
    assert rope(**KV, v_cache=24 * MB + 2 * at, ks=ks, vs=vs) == _lib.HXM_NO_DEVICE, \
        hxm.last_error()


@no_gpu
def test_rope_append_spans_past_64_bits():
    far = (1 << 40, 1 << 40, 1 << 40)
    one = dict(pages=1, page_size=1 << 30, heads=1, ks=far, vs=far)
    assert rope(**one, k=(18 * MB, 64, 64), v=(19 * MB, 64, 64)) == _lib.HXM_NO_DEVICE
    _refused(rope(**one, v_cache=24 * MB), INVALID, "keys and values")


@pytest.mark.parametrize("shape, order", [((4, 3, 8), (1, 0, 2)), ((2, 5, 3, 16), (2, 0, 1, 3)),
                                          ((4, 3, 8), (0, 1, 2)), ((8,), (0,)), ((0, 3, 8), (1, 0, 2))])
def test_new_outputs_of_permuted_rows(shape, order):
    """The output that a row operator makes itself has evenly strided rows, whatever
    the order of its input's dimensions."""
    x = torch.zeros(shape, dtype=torch.float16).permute(order)
    out, rows = hxm.ops._rows_out(None, x, shape[-1])
    assert out.shape == x.shape and out.dtype == x.dtype
    assert rows.data_ptr() == out.data_ptr() and rows.shape == (x.numel() // shape[-1], shape[-1])


@no_gpu
def test_paged_attention_refuses_more_workgroups_than_a_launch_holds():
    """2^32 - 1 work-items, 256 to a sequence and head, and 768 workgroups for the pieces of
    sequences that are cut."""
    most = (2 ** 32 - 1) // 256
    one = dict(q_heads=1, heads=1, ks=(1024, 1024, 64), vs=(1024, 1024, 64), q=(16 * MB, 64, 64),
               out=(1 << 40, 64, 64))
    assert attention(**one, batch=most) == _lib.HXM_NO_DEVICE
    _refused(attention(**one, batch=most + 1), SHAPE)
    two = dict(heads=1, ks=(1024, 1024, 64), vs=(1024, 1024, 64), q_heads=16, q=(16 * MB, 1024, 64),
               out=(1 << 40, 1024, 64))
    assert attention(**two, batch=1 << 20) == _lib.HXM_NO_DEVICE   # sixteen heads share one
    wide = dict(q_heads=65535, heads=65535, ks=(65535 * 1024, 1024, 64), vs=(65535 * 1024, 1024, 64),
                q=(16 * MB, 65535 * 64, 64), out=(1 << 40, 65535 * 64, 64))
    assert attention(**wide, batch=255) == _lib.HXM_NO_DEVICE
    _refused(attention(**wide, batch=256), SHAPE)
