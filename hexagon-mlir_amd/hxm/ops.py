"""Torch-facing host mirror of the reference's operator surface for this path.

The reference launches Triton kernels whose meaning is ``linalg.matmul`` /
row reductions and checks them against torch (``torch.matmul``,
``F.softmax``, ``F.rms_norm``, ``F.layer_norm``: test/python/triton/
test_matmul.py:86-88, test_softmax.py:91, test_rms_norm.py:84,
test_layer_norm.py).  These functions keep those names and argument meanings
and run the gfx950 kernels through the C ABI.  Tensors must already live on
the GPU; a CPU tensor is an error, never a silent fallback.
"""
from __future__ import annotations

import functools
from typing import Optional, Sequence

import torch

from ._lib import (B_KN, B_NK, BF16, F16, F32, I8, I32, IMAGE_GEMM, IMAGE_W8A16, NORM_LAYER,
                   HEAD_NORM, HEADS, KV_CACHE, NORM_NONE, NORM_RMS, OP_W8A16, OP_W8A16_SWIGLU,
                   ROW_NORM, W_NK, W_PACKED, GemmConfig, HxmError, check, lib)

_DT = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32,
       torch.int8: I8, torch.int32: I32}


def _code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


# The current device's current stream as a raw handle.  Building the Stream
# object that torch.cuda.current_stream() returns takes 2.7 us, a quarter of a
# small call's host time; the handle alone 0.1 us.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _mat(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.is_cuda and t.dim() == 2 and t.stride(1) == 1:
        return t
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (got {t.device})")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D (got {tuple(t.shape)})")
    raise ValueError(f"{name} must have a contiguous last dimension")


def _out(out: torch.Tensor, shape, dtypes, like: torch.Tensor, name: str = "out") -> torch.Tensor:
    """A caller-supplied output: a GPU matrix of exactly ``shape``, one of
    ``dtypes``, on ``like``'s device.  The C entries write shape[0] rows of
    shape[1] elements at its pointer and cannot see the allocation, so a
    wrong shape or dtype here would be a write past the tensor."""
    _mat(out, name)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)} (got {tuple(out.shape)})")
    if out.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)} (got {out.dtype})")
    if out.device != like.device:
        raise ValueError(f"{name} must be on {like.device} (got {out.device})")
    return out


def _dtype(t: torch.Tensor, dtypes, name: str) -> torch.Tensor:
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)} (got {t.dtype})")
    return t


def _vec(t: torch.Tensor, n: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    """A per-channel vector of n elements of dtype on the GPU, contiguous."""
    if not t.is_cuda or t.dtype != dtype or t.numel() != n:
        raise ValueError(f"{name} must be a GPU {dtype} tensor of {n} elements "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t if t.is_contiguous() else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))


def _b_extent(A: torch.Tensor, B: torch.Tensor, b_layout: str) -> int:
    """N of C = A @ B for B [K, N] (``"kn"``) or the [N, K] image (``"nk"``),
    after checking that B's K matches A's."""
    if b_layout not in ("kn", "nk"):
        raise ValueError(f"b_layout must be 'kn' or 'nk' (got {b_layout!r})")
    K = A.shape[1]
    kb, n = (B.shape[0], B.shape[1]) if b_layout == "kn" else (B.shape[1], B.shape[0])
    if kb != K:
        raise ValueError(f"shape mismatch A{tuple(A.shape)} B{tuple(B.shape)} ({b_layout})")
    return n


_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _config(config):
    """The C argument of a config (None: the library's choice)."""
    return None if config is None else _ptr_or_none(_cfg(config))


def _cfg(config) -> Optional[GemmConfig]:
    if config is None:
        return None
    if isinstance(config, GemmConfig):
        return config
    return GemmConfig(*config)


def _ptr_or_none(cfg):
    import ctypes
    return None if cfg is None else ctypes.byref(cfg)


def matmul(A: torch.Tensor, B: torch.Tensor, out: Optional[torch.Tensor] = None, *,
           b_layout: str = "kn", accumulate: bool = False,
           out_dtype: Optional[torch.dtype] = None, config=None, stream=None) -> torch.Tensor:
    """C = [C +] A @ B on f16/bf16/f32 with fp32 accumulation (linalg.matmul).
    f32 operands are quantised to fp16 by a pack pass (x + 0.0 then round to
    nearest even, the reference's f32 pack) and multiplied on the fp16 MFMA.

    ``b_layout="kn"``: B is [K, N] (packed per call); ``"nk"``: B is the
    resident [N, K] image from :func:`prepack_weight`."""
    _mat(A, "A"), _mat(B, "B")
    if A.dtype != B.dtype:
        raise TypeError(f"A and B must share a dtype (got {A.dtype} and {B.dtype})")
    M, K = A.shape
    N = _b_extent(A, B, b_layout)
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs out")
        out = torch.empty((M, N), dtype=out_dtype or A.dtype, device=A.device)
        if out.dtype not in _FLOATS:
            _out(out, (M, N), _FLOATS, A)
    else:
        _out(out, (M, N), _FLOATS, A)
    st = lib.hxm_matmul(A.data_ptr(), _ld(A), B.data_ptr(), _ld(B),
                        B_KN if b_layout == "kn" else B_NK, out.data_ptr(), _ld(out),
                        M, N, K, _code(A), _code(out), int(accumulate), _config(config),
                        _stream(stream))
    if st:
        check(st, "hxm_matmul")
    return out


_PLAN = {0: "mfma-full", 1: "mfma-tail", -1: "refused"}
_SOURCE = {0: "default", 1: "tuned", 2: "caller"}


def _plan_dict(p) -> dict:
    return {"op": p.op, "plan": _PLAN.get(p.plan, str(p.plan)),
            "reason": lib.hxm_reason_string(p.reason).decode(),
            "source": _SOURCE.get(p.source, str(p.source)), "config": p.config.as_tuple(),
            "k_slices": p.k_slices, "threads": p.threads, "tiles": p.tiles,
            "lds_bytes": p.lds_bytes, "workspace_bytes": p.workspace_bytes,
            "shape": (p.m, p.n, p.k)}


def plan_matmul(M: int, N: int, K: int, dtype: torch.dtype,
                out_dtype: Optional[torch.dtype] = None, *, b_layout: str = "nk",
                config=None) -> dict:
    """What a matmul call of this shape would run and why, without launching
    (hxm_plan_matmul): plan "mfma-full" / "mfma-tail" / "refused", the
    manifest-style reason, the config and where it came from, the K split,
    tiles, LDS and library workspace bytes.  A refusal is reported, not
    raised."""
    import ctypes
    from ._lib import Plan
    p = Plan()
    od = out_dtype or (torch.int32 if dtype == torch.int8 else dtype)
    cfg = _cfg(config)
    lib.hxm_plan_matmul(M, N, K, _DT[dtype], _DT[dtype], _DT[od],
                        B_KN if b_layout == "kn" else B_NK, _ptr_or_none(cfg), ctypes.byref(p))
    return _plan_dict(p)


def last_plan() -> Optional[dict]:
    """The plan of this thread's last matmul / GEMM call (hxm_last_plan)."""
    import ctypes
    from ._lib import Plan
    p = Plan()
    return _plan_dict(p) if lib.hxm_last_plan(ctypes.byref(p)) else None


def gemm_i8(A: torch.Tensor, B: torch.Tensor, out: Optional[torch.Tensor] = None, *,
            b_layout: str = "kn", accumulate: bool = False, config=None,
            stream=None) -> torch.Tensor:
    """int32 C = [C +] A @ B, exact (the reference's int8 linalg.matmul)."""
    _mat(A, "A"), _mat(B, "B")
    _dtype(A, (torch.int8,), "A"), _dtype(B, (torch.int8,), "B")
    M, K = A.shape
    N = _b_extent(A, B, b_layout)
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs out")
        out = torch.empty((M, N), dtype=torch.int32, device=A.device)
    else:
        _out(out, (M, N), (torch.int32,), A)
    st = lib.hxm_gemm_i8(A.data_ptr(), _ld(A), B.data_ptr(), _ld(B),
                         B_KN if b_layout == "kn" else B_NK, out.data_ptr(), _ld(out),
                         M, N, K, int(accumulate), _config(config), _stream(stream))
    if st:
        check(st, "hxm_gemm_i8")
    return out


def gemm_i8_dequant(A: torch.Tensor, B: torch.Tensor, row_scale: torch.Tensor,
                    col_scale: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                    b_layout: str = "kn", config=None, stream=None) -> torch.Tensor:
    """f16 C = f16(((float)(A @ B) * row_scale[:,None]) * col_scale[None,:])."""
    _mat(A, "A"), _mat(B, "B")
    _dtype(A, (torch.int8,), "A"), _dtype(B, (torch.int8,), "B")
    M, K = A.shape
    N = _b_extent(A, B, b_layout)
    if row_scale.dtype != torch.float32 or col_scale.dtype != torch.float32:
        raise TypeError("scales must be float32")
    if row_scale.numel() != M or col_scale.numel() != N:
        raise ValueError("scale lengths must be M and N")
    row_scale = _vec(row_scale, M, torch.float32, "row_scale")
    col_scale = _vec(col_scale, N, torch.float32, "col_scale")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    else:
        _out(out, (M, N), (torch.float16,), A)
    st = lib.hxm_gemm_i8_dequant(A.data_ptr(), _ld(A), B.data_ptr(), _ld(B),
                                 B_KN if b_layout == "kn" else B_NK,
                                 row_scale.data_ptr(), col_scale.data_ptr(),
                                 out.data_ptr(), _ld(out),
                                 M, N, K, _config(config), _stream(stream))
    if st:
        check(st, "hxm_gemm_i8_dequant")
    return out


def prepack_weight(B: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                   stream=None) -> torch.Tensor:
    """[K, N] -> resident [N, K] image (hmx_weight_prepack's role).  Without
    ``out`` the image is a [N, K] view of rows padded to 128 bytes (its
    stride(0) is the row stride to pass as ldb), so every row starts on a
    cache line: int8 4000^3 + dequant ran 59.5 us on 4000-byte rows and
    56.7 us on 4096-byte ones."""
    _mat(B, "B")
    K, N = B.shape
    if out is None:
        eb = B.element_size()
        kp = -(-K * eb // 128) * 128 // eb
        out = torch.empty((N, kp), dtype=B.dtype, device=B.device)[:, :K]
    _out(out, (N, K), (B.dtype,), B)
    st = lib.hxm_prepack_weight(B.data_ptr(), _ld(B), out.data_ptr(), _ld(out), K, N,
                                _code(B), _stream(stream))
    check(st, "hxm_prepack_weight")
    return out


def prepack_w8a16(W: torch.Tensor, *, stream=None) -> torch.Tensor:
    """int8 W [N, K] -> the resident GEMV image (flat int8 tensor; each
    weight in offset binary, byte = w ^ 0x80)."""
    _mat(W, "W")
    N, K = W.shape
    out = torch.empty(int(lib.hxm_w8a16_packed_bytes(N, K)), dtype=torch.int8, device=W.device)
    st = lib.hxm_prepack_w8a16(W.data_ptr(), _ld(W), N, K, out.data_ptr(), out.numel(),
                               _stream(stream))
    check(st, "hxm_prepack_w8a16")
    return out


def gemv_w8a16(x: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
               out: Optional[torch.Tensor] = None, *, N: Optional[int] = None,
               stream=None) -> torch.Tensor:
    """y = f16((x @ W.T in fp32) * scale) for int8 W [N, K] and f16 x [M, K].

    W may also be the flat image from :func:`prepack_w8a16`; then N is taken
    from ``scale`` (or passed explicitly)."""
    _mat(x, "x")
    _dtype(x, (torch.float16,), "x"), _dtype(W, (torch.int8,), "W")
    M, K = x.shape
    packed = W.dim() == 1
    if packed:
        if not W.is_cuda:
            raise ValueError(f"W must be a GPU tensor (got {W.device})")
        N = scale.numel() if N is None else N
        if W.numel() < lib.hxm_w8a16_packed_bytes(N, K):
            raise ValueError("packed image too small for [N, K]")
        ldw = K
    else:
        _mat(W, "W")
        N = W.shape[0]
        if W.shape[1] != K:
            raise ValueError("W must be [N, K]")
        ldw = _ld(W)
    scale = _vec(scale, N, torch.float16, "scale")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=x.device)
    else:
        _out(out, (M, N), (torch.float16,), x)
    st = lib.hxm_gemv_w8a16(x.data_ptr(), _ld(x), W.data_ptr(), ldw,
                            W_PACKED if packed else W_NK, scale.data_ptr(),
                            out.data_ptr(), _ld(out), M, N, K, _stream(stream))
    if st:
        check(st, "hxm_gemv_w8a16")
    return out


def _f32_vec(t: torch.Tensor, n: int, name: str) -> torch.Tensor:
    if not t.is_cuda or t.dtype != torch.float32 or t.numel() != n:
        raise ValueError(f"{name} must be a GPU float32 tensor of {n} elements")
    return t.contiguous()


def gemm_w8a16(x: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
               out: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
               config=None, stream=None) -> torch.Tensor:
    """y = f16((x @ W.T in fp32) * scale) for f16 x [M, K], int8 W [N, K] and
    fp32 per-channel scale [N] (the large-M W8A16 GEMM of the FFN).  With an
    f16 ``residual`` [M, N]: y = f16(fp32((x @ W.T) * scale) + residual)
    (hxm_gemm_w8a16_residual); ``out`` may be ``residual`` itself."""
    _mat(x, "x"), _mat(W, "W")
    _dtype(x, (torch.float16,), "x"), _dtype(W, (torch.int8,), "W")
    M, K = x.shape
    N = W.shape[0]
    if W.shape[1] != K:
        raise ValueError("W must be [N, K]")
    scale = _f32_vec(scale, N, "scale")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=x.device)
    else:
        _out(out, (M, N), (torch.float16,), x)
    if residual is not None:
        _mat(residual, "residual")
        if tuple(residual.shape) != (M, N) or residual.dtype != torch.float16:
            raise ValueError(f"residual must be f16 [{M}, {N}]")
        st = lib.hxm_gemm_w8a16_residual(x.data_ptr(), _ld(x), W.data_ptr(), _ld(W),
                                         scale.data_ptr(), residual.data_ptr(), _ld(residual),
                                         out.data_ptr(), _ld(out), M, N, K, _config(config),
                                         _stream(stream))
        if st:
            check(st, "hxm_gemm_w8a16_residual")
        return out
    st = lib.hxm_gemm_w8a16(x.data_ptr(), _ld(x), W.data_ptr(), _ld(W), scale.data_ptr(),
                            out.data_ptr(), _ld(out), M, N, K, _config(config),
                            _stream(stream))
    if st:
        check(st, "hxm_gemm_w8a16")
    return out


def swiglu_pack(Wg: torch.Tensor, Wu: torch.Tensor, gate_scale: torch.Tensor,
                up_scale: torch.Tensor, *, stream=None):
    """The fused gate/up image (int8 [128*ceil(I/64), K], each weight stored
    in offset binary, byte = w ^ 0x80) and its fp32 scales from gate/up
    weights int8 [I, K] and fp32 scales [I]; made once per weight pair."""
    _mat(Wg, "Wg"), _mat(Wu, "Wu")
    I, K = Wg.shape
    if tuple(Wu.shape) != (I, K) or _ld(Wu) != _ld(Wg):
        raise ValueError("Wg and Wu must both be [I, K] with the same row stride")
    sg = _f32_vec(gate_scale, I, "gate_scale")
    su = _f32_vec(up_scale, I, "up_scale")
    rows = lib.hxm_swiglu_packed_rows(I)
    Wgu = torch.empty((rows, K), dtype=torch.int8, device=Wg.device)
    sgu = torch.empty(rows, dtype=torch.float32, device=Wg.device)
    st = lib.hxm_swiglu_pack(Wg.data_ptr(), Wu.data_ptr(), _ld(Wg), sg.data_ptr(),
                             su.data_ptr(), I, K, Wgu.data_ptr(), sgu.data_ptr(),
                             _stream(stream))
    check(st, "hxm_swiglu_pack")
    return Wgu, sgu


def gemm_w8a16_swiglu(x: torch.Tensor, Wgu: torch.Tensor, sgu: torch.Tensor, I: int,
                      out: Optional[torch.Tensor] = None, *, config=None,
                      stream=None) -> torch.Tensor:
    """h = f16(silu(x @ Wg.T * sg) * (x @ Wu.T * su)) from the
    :func:`swiglu_pack` image; h is [M, I]."""
    _mat(x, "x"), _mat(Wgu, "Wgu")
    _dtype(x, (torch.float16,), "x"), _dtype(Wgu, (torch.int8,), "Wgu")
    M, K = x.shape
    rows = lib.hxm_swiglu_packed_rows(I)
    if tuple(Wgu.shape) != (rows, K) or _ld(Wgu) != K:
        raise ValueError(f"Wgu must be the contiguous [{rows}, {K}] swiglu_pack image")
    sgu = _f32_vec(sgu, rows, "sgu")
    if out is None:
        out = torch.empty((M, I), dtype=torch.float16, device=x.device)
    else:
        _out(out, (M, I), (torch.float16,), x)
    st = lib.hxm_gemm_w8a16_swiglu(x.data_ptr(), _ld(x), Wgu.data_ptr(), sgu.data_ptr(),
                                   out.data_ptr(), _ld(out), M, I, K, _config(config),
                                   _stream(stream))
    if st:
        check(st, "hxm_gemm_w8a16_swiglu")
    return out


def swiglu_ffn(x: torch.Tensor, gamma: torch.Tensor, Wgu: torch.Tensor, sgu: torch.Tensor,
               Wd: torch.Tensor, sd: torch.Tensor, I: int, *, eps: float = 1e-6,
               residual: bool = False, configs=(None, None), stream=None) -> torch.Tensor:
    """The Llama-style SwiGLU FFN block: RMSNorm -> fused gate/up GEMM with
    SiLU * mul -> down GEMM.  x f16 [T, H]; gamma f16 [H]; Wgu/sgu from
    :func:`swiglu_pack`; Wd int8 [H, I] with fp32 scales sd [H].  With
    ``residual`` the down GEMM's epilogue adds x: the block returns
    x + FFN(x)."""
    xn = rms_norm(x, (x.shape[-1],), gamma, eps=eps, stream=stream)
    h = gemm_w8a16_swiglu(xn, Wgu, sgu, I, config=configs[0], stream=stream)
    return gemm_w8a16(h, Wd, sd, residual=x if residual else None, config=configs[1],
                      stream=stream)


def w8a16_configs(swiglu: bool = False):
    """The compiled W8A16 GEMM configurations (bk in f16 elements)."""
    n = lib.hxm_w8a16_configs(int(swiglu), None, 0)
    arr = (GemmConfig * n)()
    lib.hxm_w8a16_configs(int(swiglu), arr, n)
    return list(arr)


def tune_w8a16(x: torch.Tensor, W: torch.Tensor, scale: torch.Tensor, out: torch.Tensor, *,
               swiglu: bool = False, reps: int = 5, stream=None):
    """Measured tile search for :func:`gemm_w8a16` (W [N, K], scale [N]) or,
    with swiglu=True, :func:`gemm_w8a16_swiglu` (W = Wgu, scale = sgu, out
    [M, I]).  The winner is cached for later calls; returns (GemmConfig,
    report dict).  reps=0 calibrates the repetitions per config as in
    :func:`tune_gemm`; the int8-weight configs are not priced, so all run."""
    import ctypes
    import json
    _mat(x, "x"), _mat(W, "W")
    _dtype(x, (torch.float16,), "x"), _dtype(W, (torch.int8,), "W")
    M, K = x.shape
    if swiglu:
        N = out.shape[1]
        rows = lib.hxm_swiglu_packed_rows(N)
        if tuple(W.shape) != (rows, K) or _ld(W) != K:
            raise ValueError(f"W must be the contiguous [{rows}, {K}] swiglu_pack image")
        scale = _f32_vec(scale, rows, "scale")
    else:
        N = W.shape[0]
        if W.shape[1] != K:
            raise ValueError("W must be [N, K]")
        scale = _f32_vec(scale, N, "scale")
    _out(out, (M, N), (torch.float16,), x)
    best = GemmConfig()
    buf = ctypes.create_string_buffer(1 << 16)
    st = lib.hxm_tune_w8a16(OP_W8A16_SWIGLU if swiglu else OP_W8A16, x.data_ptr(), _ld(x),
                            W.data_ptr(), _ld(W), scale.data_ptr(),
                            out.data_ptr(), _ld(out), M, N, K, reps, ctypes.byref(best), buf,
                            len(buf), _stream(stream))
    check(st, "hxm_tune_w8a16")
    return best, json.loads(buf.value.decode())


class _DeviceArray:
    """A non-owning view of library-owned device memory for torch.as_tensor
    (the CUDA array interface, which the ROCm build of torch accepts)."""

    _TYPESTR = {I8: "|i1", F16: "<f2", BF16: "<V2", F32: "<f4"}

    def __init__(self, ptr: int, shape, dtype_code: int):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "data": (ptr, False),
                                         "typestr": self._TYPESTR[dtype_code], "version": 3,
                                         "strides": None}


def resident_weight(W: torch.Tensor, kind: str = "gemm", *, expect_dtype=None,
                    expect_shape=None, stream=None) -> torch.Tensor:
    """The content-addressed resident image of a weight, packed on first use
    (WeightPrepack.pack, hmx_weight_prepack.py:124-168).

    ``kind="gemm"``: W is B [K, N] (int8/f16/bf16, or f32 -> an f16 image);
    returns the [N, K] image for ``b_layout="nk"``.  ``kind="w8a16"``: W is
    int8 [N, K]; returns the flat packed GEMV image.  The returned tensor
    views library-owned memory that stays valid until ``hxm_release_cache``.
    ``expect_dtype`` / ``expect_shape`` are the contract: a mismatch raises."""
    import ctypes
    _mat(W, "W")
    rows, cols = W.shape
    k = {"gemm": IMAGE_GEMM, "w8a16": IMAGE_W8A16}[kind]
    exp_dt = -1 if expect_dtype is None else _DT[expect_dtype]
    shp = None if expect_shape is None else (ctypes.c_int64 * 2)(*expect_shape)
    img = ctypes.c_void_p()
    img_dt = ctypes.c_int32()
    st = lib.hxm_resident_weight(W.data_ptr(), _ld(W), rows, cols, _code(W), exp_dt, shp, k,
                                 ctypes.byref(img), ctypes.byref(img_dt), _stream(stream))
    check(st, "hxm_resident_weight")
    if k == IMAGE_GEMM:
        if img_dt.value == BF16:   # no bf16 typestr: view the bits, then reinterpret
            t = torch.as_tensor(_DeviceArray(img.value, (cols, rows), F16), device=W.device)
            return t.view(torch.bfloat16)
        return torch.as_tensor(_DeviceArray(img.value, (cols, rows), img_dt.value),
                               device=W.device)
    nbytes = lib.hxm_w8a16_packed_bytes(rows, cols)
    return torch.as_tensor(_DeviceArray(img.value, (nbytes,), I8), device=W.device)


def _rows(x: torch.Tensor):
    if not x.is_cuda:
        raise ValueError(f"x must be a GPU tensor (got {x.device})")
    if x.stride(-1) != 1:
        raise ValueError("x must have a contiguous last dimension")
    if x.dim() == 2:
        return x, x.shape[0], x.shape[1]
    cols = x.shape[-1]
    x2 = x.reshape(-1, cols)
    return x2, x2.shape[0], cols


def _rows_out(out: Optional[torch.Tensor], x: torch.Tensor, cols: int):
    """The output of a row op: new, or the caller's of x's shape and dtype
    (rows of it may be strided, its last dimension contiguous)."""
    if out is None:
        if x.dim() == 2:
            out = torch.empty_like(x)
            return out, out
        # Not x's own strides: its dimensions may be permuted.
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif tuple(out.shape) != tuple(x.shape) or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"out must be {x.dtype} {tuple(x.shape)} on {x.device} "
                         f"(got {out.dtype} {tuple(out.shape)} on {out.device})")
    elif out.stride(-1) != 1:
        raise ValueError("out must have a contiguous last dimension")
    try:
        return out, out.view(-1, cols)   # a view: the kernel writes into out itself
    except RuntimeError:
        raise ValueError("out's rows must be evenly strided (viewable as [rows, cols])") from None


def _row_param(t: Optional[torch.Tensor], x: torch.Tensor, cols: int, name: str):
    """gamma / beta: None, or [cols] of x's dtype on x's device."""
    if t is None:
        return None
    if t.numel() != cols or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must be {x.dtype} [{cols}] on {x.device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t.contiguous()


def softmax(x: torch.Tensor, dim: int = -1, out: Optional[torch.Tensor] = None, *,
            stream=None) -> torch.Tensor:
    """Row softmax over the last dimension (F.softmax(x, dim=-1))."""
    if dim not in (-1, x.dim() - 1):
        raise ValueError("only the last dimension is supported")
    x2, rows, cols = _rows(x)
    out, o2 = _rows_out(out, x, cols)
    st = lib.hxm_softmax_rows(x2.data_ptr(), _ld(x2), o2.data_ptr(), _ld(o2), rows, cols,
                              _code(x), _stream(stream))
    if st:
        check(st, "hxm_softmax_rows")
    return out


def rms_norm(x: torch.Tensor, normalized_shape: Sequence[int],
             weight: Optional[torch.Tensor] = None, eps: Optional[float] = None,
             out: Optional[torch.Tensor] = None, *, stream=None) -> torch.Tensor:
    """F.rms_norm over the last dimension."""
    x2, rows, cols = _rows(x)
    if tuple(normalized_shape) != (cols,):
        raise ValueError("normalized_shape must be (x.shape[-1],)")
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    out, o2 = _rows_out(out, x, cols)
    weight = _row_param(weight, x, cols, "weight")
    st = lib.hxm_rmsnorm_rows(x2.data_ptr(), _ld(x2),
                              None if weight is None else weight.data_ptr(), o2.data_ptr(), _ld(o2),
                              rows, cols, float(eps), _code(x), _stream(stream))
    if st:
        check(st, "hxm_rmsnorm_rows")
    return out


def layer_norm(x: torch.Tensor, normalized_shape: Sequence[int],
               weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, *,
               return_stats: bool = False, stream=None):
    """F.layer_norm over the last dimension; optionally returns (y, mean, rstd)."""
    x2, rows, cols = _rows(x)
    if tuple(normalized_shape) != (cols,):
        raise ValueError("normalized_shape must be (x.shape[-1],)")
    out, o2 = _rows_out(out, x, cols)
    weight = _row_param(weight, x, cols, "weight")
    bias = _row_param(bias, x, cols, "bias")
    mean = rstd = None
    if return_stats:
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    st = lib.hxm_layernorm_rows(
        x2.data_ptr(), _ld(x2), None if weight is None else weight.data_ptr(),
        None if bias is None else bias.data_ptr(), o2.data_ptr(), _ld(o2),
        None if mean is None else mean.data_ptr(), None if rstd is None else rstd.data_ptr(),
        rows, cols, float(eps), _code(x), _stream(stream))
    if st:
        check(st, "hxm_layernorm_rows")
    return (out, mean, rstd) if return_stats else out


# The current device's number, without the Python around torch.cuda.current_device().
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _on_current(t: torch.Tensor, name: str) -> int:
    """The device of a GPU tensor, which must be the current one (the
    decoder-layer operators launch there)."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (got {t.device})")
    dev = t.get_device()
    if dev != _current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is "
                         f"cuda:{_current_device()}")
    return dev


def _tensor(t: torch.Tensor, dtype: torch.dtype, shape, dev: int, name: str) -> torch.Tensor:
    """t, checked to be of this dtype and shape on this device."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on cuda:{dev} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t


def _ints(t: torch.Tensor, shape, dev: int, name: str) -> int:
    """The address of a contiguous int32 tensor of this shape on this device."""
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be torch.int32 (got {t.dtype})")
    if t.shape != shape or t.get_device() != dev:
        _tensor(t, torch.int32, shape, dev, name)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _on_stream(op):
    """An operator whose outputs and contiguous copies belong to the stream it runs on:
    with ``stream`` given, the whole call is made with that stream the current one."""
    @functools.wraps(op)
    def call(*args, stream=None, **kwargs):
        if stream is None:
            return op(*args, **kwargs)
        with torch.cuda.stream(stream):
            return op(*args, **kwargs)
    return call


def _current_stream(dev: int) -> int:
    """_stream() for a device known to be the current one."""
    return _raw_stream(dev) if _raw_stream is not None else _stream()


def _row_ld(t: torch.Tensor, rows: int, cols: int) -> int:
    """The leading dimension of a [rows, cols] view; one row has none."""
    return t.stride(0) if rows > 1 else cols


def _param(t: Optional[torch.Tensor], dtype: torch.dtype, cols: int, dev: int, name: str,
           what: str):
    """(contiguous t, its address): [cols] of dtype on this device, or None."""
    if t is None:
        return None, 0
    if t.numel() != cols or t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name}_{what} must be {dtype} [{cols}] on cuda:{dev} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    t = t.contiguous()
    return t, t.data_ptr()


_NORMS = {"none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}


def _row_norm(kind: str, weight, bias, eps: float, dtype: torch.dtype, cols: int, dev: int,
              name: str):
    """The hxm_row_norm, and the tensors it points to (to be kept until the call)."""
    if kind not in _NORMS:
        raise ValueError(f"{name} must be one of {sorted(_NORMS)} (got {kind!r})")
    w, w_ptr = _param(weight, dtype, cols, dev, name, "weight")
    b, b_ptr = _param(bias, dtype, cols, dev, name, "bias")
    return ROW_NORM.pack(_NORMS[kind], eps, w_ptr, b_ptr), w, b


@_on_stream
def residual_norm(h: torch.Tensor, x: torch.Tensor, *, post: str = "none",
                  post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, post_eps: float = 1e-6,
                  pre: str = "rms", pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, pre_eps: float = 1e-6,
                  gate: Optional[torch.Tensor] = None, block_scale: float = 1.0,
                  residual_scale: float = 1.0, out: Optional[torch.Tensor] = None,
                  normed_out: Optional[torch.Tensor] = None):
    """The norms around a block fused with its gate and the residual
    (hxm_residual_norm_rows): returns (y, z),

        y = residual_scale * x + block_scale * gate * post(h)
        z = pre(y)

    for the block's output ``h`` and the residual stream ``x`` (same shape and
    dtype).  ``post`` / ``pre``: "none", "rms" or "layer", with weights and
    biases [cols]; ``pre="none"`` gives z = None.  ``gate``: [cols], or
    [G, cols] with one row for every rows / G consecutive rows.  ``out`` (y)
    and ``normed_out`` (z) may be ``x`` or ``h`` themselves."""
    dev = _on_current(h, "h")
    dtype, shape = h.dtype, h.shape
    if dtype not in _FLOATS:
        raise TypeError(f"h must be {' or '.join(str(d) for d in _FLOATS)} (got {dtype})")
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"h must have a last dimension of one element or more "
                         f"(got {tuple(shape)})")
    _tensor(x, dtype, shape, dev, "x")
    h2, rows, cols = _rows(h)
    x2, _, _ = _rows(x)
    y, y2 = _rows_out(out, h, cols)
    if pre == "none":
        if normed_out is not None:
            raise ValueError("normed_out needs a pre norm")
        z = None
        z_ptr, ldz = None, 0
    else:
        z, z2 = _rows_out(normed_out, h, cols)
        z_ptr, ldz = z2.data_ptr(), _row_ld(z2, rows, cols)
    post_n, post_w, post_b = _row_norm(post, post_weight, post_bias, post_eps, dtype, cols, dev,
                                       "post")
    pre_n, pre_w, pre_b = _row_norm(pre, pre_weight, pre_bias, pre_eps, dtype, cols, dev, "pre")
    gate_ptr, ldg, G = None, 0, 0
    if gate is not None:
        if gate.dtype != dtype or gate.get_device() != dev:
            raise ValueError(f"gate must be {dtype} on cuda:{dev} "
                             f"(got {gate.dtype} on {gate.device})")
        g2 = gate.view(1, -1) if gate.dim() == 1 else gate
        if g2.dim() != 2 or g2.shape[1] != cols or g2.shape[0] < 1 or rows % g2.shape[0]:
            raise ValueError(f"gate must be [{cols}] or [G, {cols}] with G dividing {rows} rows "
                             f"(got {tuple(gate.shape)})")
        gate = g2 if g2.stride(1) == 1 else g2.contiguous()
        gate_ptr, ldg, G = gate.data_ptr(), _ld(gate), gate.shape[0]
    st = lib.hxm_residual_norm_rows(h2.data_ptr(), _row_ld(h2, rows, cols), x2.data_ptr(),
                                    _row_ld(x2, rows, cols), post_n, gate_ptr, ldg, G,
                                    block_scale, residual_scale, pre_n, y2.data_ptr(),
                                    _row_ld(y2, rows, cols), z_ptr, ldz, rows, cols, _DT[dtype],
                                    _current_stream(dev))
    if st:
        check(st, "hxm_residual_norm_rows")
    return y, z


_HALVES = (torch.float16, torch.bfloat16)


def _heads(t: torch.Tensor, dtype: torch.dtype, shape, dev: int, name: str) -> bytes:
    """The hxm_heads of a [tokens, heads, dim] tensor."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != dev:
        _tensor(t, dtype, shape, dev, name)
    ts, hs, inner = t.stride()
    if inner != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    return HEADS.pack(t.data_ptr(), ts, hs)


def _kv_cache(k: torch.Tensor, v: torch.Tensor):
    """The hxm_kv_cache of [pages, heads, page_size, dim] tensors of any strides
    (a cache that keeps tokens before heads is passed transposed), its heads
    and dim, dtype and device."""
    dev = _on_current(k, "k_cache")
    dtype, shape = k.dtype, k.shape
    if len(shape) != 4:
        raise ValueError(f"k_cache must be [pages, heads, page_size, dim] (got {tuple(shape)})")
    if dtype not in _HALVES:
        raise TypeError(f"k_cache must be {' or '.join(str(d) for d in _HALVES)} (got {dtype})")
    _tensor(v, dtype, shape, dev, "v_cache")
    pages, heads, page, dim = shape
    kp, kh, kt, ki = k.stride()
    vp, vh, vt, vi = v.stride()
    if ki != 1 or vi != 1:
        raise ValueError("k_cache and v_cache must have a contiguous last dimension")
    return (KV_CACHE.pack(k.data_ptr(), v.data_ptr(), pages, page, heads, dim, kp, kh, kt, vp, vh,
                          vt), heads, dim, dtype, dev)


@_on_stream
def rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                positions: Optional[torch.Tensor] = None,
                cos_sin: Optional[torch.Tensor] = None, *, interleaved: bool = False,
                q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotary positions and the append to a paged cache in one launch
    (hxm_rope_append): returns the rotated q and stores the rotated k and v.

    q [T, Hq, D] (or None), k and v [T, Hkv, D] f16 / bf16, the last dimension
    contiguous (heads of a fused projection's output are fine); the caches
    [pages, Hkv, page_size, D], any strides; ``slots`` int32 [T]: page *
    page_size + offset, all different, -1 for a row that stores nothing.
    ``positions`` int32 [T] and ``cos_sin`` fp32 [max_pos, rot_dim] (cosines,
    then sines) rotate the first rot_dim dims, in halves or (``interleaved``)
    in neighbouring pairs; without cos_sin nothing is rotated.  ``q_out`` may be
    q."""
    return _append("hxm_rope_append", q, k, v, k_cache, v_cache, slots, positions, cos_sin,
                   interleaved, q_out, None)


def _append(entry, q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved, q_out, norms):
    """The call of either append; norms: (kind, eps, q_weight, q_bias, k_weight, k_bias)."""
    cache, heads, dim, dtype, dev = _kv_cache(k_cache, v_cache)
    if k.dim() != 3:
        raise ValueError(f"k must be [tokens, heads, dim] (got {tuple(k.shape)})")
    T = k.shape[0]
    kh = _heads(k, dtype, (T, heads, dim), dev, "k")
    vh = _heads(v, dtype, (T, heads, dim), dev, "v")
    slot_p = _ints(slots, (T,), dev, "slots")
    pos_p = tab_p = None
    rot = ld = max_pos = 0
    if cos_sin is not None:
        if positions is None:
            raise ValueError("cos_sin needs positions")
        pos_p = _ints(positions, (T,), dev, "positions")
        _mat(cos_sin, "cos_sin")
        if cos_sin.dtype != torch.float32 or cos_sin.get_device() != dev:
            raise ValueError(f"cos_sin must be torch.float32 on cuda:{dev} "
                             f"(got {cos_sin.dtype} on {cos_sin.device})")
        max_pos, rot = cos_sin.shape
        tab_p, ld = cos_sin.data_ptr(), _ld(cos_sin)
    qh = oh = None
    hq = 0
    if q is not None:
        if q.dim() != 3:
            raise ValueError(f"q must be [tokens, heads, dim] (got {tuple(q.shape)})")
        hq = q.shape[1]
        qh = _heads(q, dtype, (T, hq, dim), dev, "q")
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        oh = _heads(q_out, dtype, (T, hq, dim), dev, "q_out")
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if norms is None:
        st = lib.hxm_rope_append(qh, oh, hq, kh, vh, pos_p, tab_p, ld, max_pos, rot,
                                 int(interleaved), slot_p, cache, T, _DT[dtype],
                                 _current_stream(dev))
    else:
        kind, eps, qw, qb, kw, kb = norms
        qn, *keep_q = _head_norm(kind, eps, qw, qb, hq, dim, dtype, dev, "q")
        kn, *keep_k = _head_norm(kind, eps, kw, kb, heads, dim, dtype, dev, "k")
        st = lib.hxm_norm_rope_append(qh, oh, hq, kh, vh, qn, kn, pos_p, tab_p, ld, max_pos, rot,
                                      int(interleaved), slot_p, cache, T, _DT[dtype],
                                      _current_stream(dev))
    if st:
        check(st, entry)
    return q_out


def _head_norm(kind: str, eps: float, weight, bias, heads: int, dim: int, dtype, dev: int,
               name: str):
    """The hxm_head_norm, and the tensors it points to (to be kept until the call)."""
    if kind not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)} (got {kind!r})")
    each = (weight is not None and weight.dim() == 2) or (bias is not None and bias.dim() == 2)
    shape = (heads, dim) if each else (dim,)
    w, w_ptr = _head_param(weight, dtype, shape, dev, name, "weight")
    b, b_ptr = _head_param(bias, dtype, shape, dev, name, "bias")
    return HEAD_NORM.pack(_NORMS[kind], eps, w_ptr, b_ptr, dim if each else 0), w, b


def _head_param(t: Optional[torch.Tensor], dtype: torch.dtype, shape, dev: int, name: str,
                what: str):
    """(contiguous t, its address): of this shape and dtype on this device, or None."""
    if t is None:
        return None, 0
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name}_{what} must be {dtype} {shape} on cuda:{dev}, [{shape[-1]}] for "
                         f"all heads or [heads, {shape[-1]}], like its other parameter "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    t = t.contiguous()
    return t, t.data_ptr()


@_on_stream
def norm_rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                     k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                     positions: Optional[torch.Tensor] = None,
                     cos_sin: Optional[torch.Tensor] = None, *, norm: str = "rms",
                     q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None,
                     q_bias: Optional[torch.Tensor] = None,
                     k_bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     interleaved: bool = False,
                     q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """:func:`rope_append` with the norm of each query and key head ("rms" or
    "layer" over its D elements) in front of the rotation, in the same pass
    (hxm_norm_rope_append).  Weights and biases of the inputs' dtype: [D] for all
    heads, or [heads, D]; without one it is 1 / 0."""
    return _append("hxm_norm_rope_append", q, k, v, k_cache, v_cache, slots, positions, cos_sin,
                   interleaved, q_out, (norm, eps, q_weight, q_bias, k_weight, k_bias))


def _block_table(t: torch.Tensor, batch: int, dev: int):
    """(address, row stride, columns) of an int32 [batch, table_pages] table."""
    _mat(t, "block_table")
    if t.dtype != torch.int32:
        raise TypeError(f"block_table must be torch.int32 (got {t.dtype})")
    rows, table_pages = t.shape
    if rows != batch or t.get_device() != dev:
        raise ValueError(f"block_table must have {batch} rows on cuda:{dev} "
                         f"(got {tuple(t.shape)} on {t.device})")
    return t.data_ptr(), _ld(t), table_pages


@_on_stream
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                    scale: Optional[float] = None, window: int = 0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of one new token per sequence over a paged cache
    (hxm_paged_attention): q [B, Hq, D] f16 / bf16 against the caches [pages,
    Hkv, page_size, D] (any strides; Hq a multiple of Hkv).  ``block_table``
    int32 [B, table_pages] names each sequence's pages in order, ``seq_lens``
    int32 [B] its tokens (the new one included; 0: the row gives zeros).
    ``scale`` defaults to D ** -0.5; ``window`` keeps the last tokens only
    (0: all).  Returns out, or (out, lse) with the fp32 [B, Hq] logarithm of
    the softmax's sum."""
    cache, _, dim, dtype, dev = _kv_cache(k_cache, v_cache)
    if q.dim() != 3:
        raise ValueError(f"q must be [batch, heads, dim] (got {tuple(q.shape)})")
    B, hq, _ = q.shape
    qh = _heads(q, dtype, (B, hq, dim), dev, "q")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    oh = _heads(out, dtype, (B, hq, dim), dev, "out")
    table_p, ld_table, table_pages = _block_table(block_table, B, dev)
    lens_p = _ints(seq_lens, (B,), dev, "seq_lens")
    lse = lse_p = None
    if return_lse:
        lse = torch.empty(B, hq, dtype=torch.float32, device=q.device)
        lse_p = lse.data_ptr()
    st = lib.hxm_paged_attention(qh, oh, hq, cache, table_p, ld_table, table_pages, lens_p, B,
                                 dim ** -0.5 if scale is None else scale, window, lse_p,
                                 _DT[dtype], _current_stream(dev))
    if st:
        check(st, "hxm_paged_attention")
    return (out, lse) if return_lse else out


@_on_stream
def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, seq_lens: torch.Tensor,
                   parents: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                   window: int = 0, out: Optional[torch.Tensor] = None,
                   return_lse: bool = False):
    """Attention of a tree of drafted tokens per sequence over a paged cache
    (hxm_tree_attention): q [B, T, Hq, D] f16 / bf16, T (up to 64) tokens of each
    sequence, which are the last of its ``seq_lens`` tokens in the caches
    (:func:`paged_attention` describes those).  ``parents`` int32 [B, T]: the
    token before each in its branch, an earlier one of the T or -1 for the
    context; -2 marks padding (zeros, -inf in lse); None is a chain.  A token
    sees the context, itself and the tokens above it, ``window`` (0: all) the
    nearest of them.  Returns out, or (out, lse) with lse fp32 [B, T, Hq]."""
    cache, _, dim, dtype, dev = _kv_cache(k_cache, v_cache)
    if q.dim() != 4:
        raise ValueError(f"q must be [batch, tokens, heads, dim] (got {tuple(q.shape)})")
    B, T, hq, _ = q.shape
    qh = _token_heads(q, dtype, (B, T, hq, dim), dev, "q")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    oh = _token_heads(out, dtype, (B, T, hq, dim), dev, "out")
    table_p, ld_table, table_pages = _block_table(block_table, B, dev)
    lens_p = _ints(seq_lens, (B,), dev, "seq_lens")
    parents_p = None if parents is None else _ints(parents, (B, T), dev, "parents")
    lse = lse_p = None
    if return_lse:
        lse = torch.empty(B, T, hq, dtype=torch.float32, device=q.device)
        lse_p = lse.data_ptr()
    st = lib.hxm_tree_attention(qh, oh, hq, cache, table_p, ld_table, table_pages, lens_p,
                                parents_p, B, T, dim ** -0.5 if scale is None else scale, window,
                                lse_p, _DT[dtype], _current_stream(dev))
    if st:
        check(st, "hxm_tree_attention")
    return (out, lse) if return_lse else out


def _token_heads(t: torch.Tensor, dtype: torch.dtype, shape, dev: int, name: str) -> bytes:
    """The hxm_heads of a [batch, tokens, heads, dim] tensor, its tokens one after the
    other over the batch."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != dev:
        _tensor(t, dtype, shape, dev, name)
    bs, ts, hs, inner = t.stride()
    if inner != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    B, T = shape[0], shape[1]
    if B > 1 and T > 1 and bs != T * ts:
        raise ValueError(f"{name}'s tokens must be evenly strided over the batch")
    return HEADS.pack(t.data_ptr(), ts if T > 1 else bs, hs)


def _tokens(t: torch.Tensor, name: str) -> torch.Tensor:
    """[batch, tokens, heads, dim] as [batch * tokens, heads, dim], without a copy."""
    try:
        return t.view(t.shape[0] * t.shape[1], *t.shape[2:])
    except RuntimeError:
        raise ValueError(f"{name}'s tokens must be evenly strided over the batch") from None


@_on_stream
def verify_draft(tokens: torch.Tensor, target: torch.Tensor, uniform: torch.Tensor,
                 parents: Optional[torch.Tensor] = None, draft: Optional[torch.Tensor] = None):
    """Which drafted tokens the target's probabilities keep, and the token that
    follows them (hxm_verify_draft, which has the rule): returns (path [B, T],
    counts [B], next_tokens [B]), int32.

    ``tokens`` int32 [B, T] (up to 64), the first the last token sampled before;
    ``parents`` as :func:`tree_attention` takes them (None: chains).  ``target``
    [B, T, V] holds the target's probabilities after each token, ``draft`` those
    that its child was drawn from (of one child each; None: children chosen
    without chance), f16, bf16 or f32; ``uniform`` fp32 [B, T] random numbers, the
    first of a sequence for the token that follows."""
    dev = _on_current(target, "target")
    if target.dim() != 3:
        raise ValueError(f"target must be [batch, tokens, vocab] (got {tuple(target.shape)})")
    B, T, V = target.shape
    dtype = target.dtype
    _dtype(target, _FLOATS, "target")
    tokens_p = _ints(tokens, (B, T), dev, "tokens")
    parents_p = None if parents is None else _ints(parents, (B, T), dev, "parents")
    if not _tensor(uniform, torch.float32, (B, T), dev, "uniform").is_contiguous():
        raise ValueError("uniform must be contiguous")
    t2 = _mat(_tokens(target, "target"), "target")
    draft_p, ldd = None, 0
    if draft is not None:
        d2 = _mat(_tokens(_tensor(draft, dtype, (B, T, V), dev, "draft"), "draft"), "draft")
        draft_p, ldd = d2.data_ptr(), _row_ld(d2, B * T, V)
    out = torch.empty(B * T + 2 * B, dtype=torch.int32, device=target.device)
    path, counts, following = out[:B * T].view(B, T), out[B * T:B * T + B], out[B * T + B:]
    at = out.data_ptr()
    st = lib.hxm_verify_draft(tokens_p, parents_p, t2.data_ptr(), _row_ld(t2, B * T, V), draft_p,
                              ldd, uniform.data_ptr(), at, at + 4 * B * T, at + 4 * B * (T + 1), B,
                              T, V, _DT[dtype], _current_stream(dev))
    if st:
        check(st, "hxm_verify_draft")
    return path, counts, following


def _kv_layers(k: torch.Tensor, v: torch.Tensor):
    """(hxm_kv_cache of the first layer, layers, their strides, dtype, device) of
    [layers, pages, heads, page_size, dim] caches, or of one layer's."""
    if k.dim() == 4:
        cache, _, _, dtype, dev = _kv_cache(k, v)
        return cache, 1, 0, 0, dtype, dev
    shape, dtype = k.shape, k.dtype
    if len(shape) != 5 or v.shape != shape or not shape[0]:
        raise ValueError("k_cache and v_cache must be [pages, heads, page_size, dim], or with a "
                         f"dimension of layers before (got {tuple(shape)}, {tuple(v.shape)})")
    dev = _on_current(k, "k_cache")
    if dtype not in _HALVES:
        raise TypeError(f"k_cache must be {' or '.join(str(d) for d in _HALVES)} (got {dtype})")
    _tensor(v, dtype, shape, dev, "v_cache")
    layers, pages, heads, page, dim = shape
    kl, kp, kh, kt, ki = k.stride()
    vl, vp, vh, vt, vi = v.stride()
    if ki != 1 or vi != 1:
        raise ValueError("k_cache and v_cache must have a contiguous last dimension")
    return (KV_CACHE.pack(k.data_ptr(), v.data_ptr(), pages, page, heads, dim, kp, kh, kt, vp, vh,
                          vt), layers, kl, vl, dtype, dev)


@_on_stream
def compact_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, path: torch.Tensor,
                  counts: torch.Tensor) -> torch.Tensor:
    """The rows of the kept tokens moved behind the context in all layers' caches
    (hxm_compact_cache): returns the sequences' new lengths, int32 [B].

    The caches are [layers, pages, Hkv, page_size, D] (or one layer's, without the
    first dimension), f16 / bf16, any strides; ``block_table`` and ``seq_lens`` as
    :func:`tree_attention` takes them, ``path`` int32 [B, T] and ``counts`` int32
    [B] as :func:`verify_draft` gives them."""
    cache, layers, kls, vls, dtype, dev = _kv_layers(k_cache, v_cache)
    if path.dim() != 2:
        raise ValueError(f"path must be [batch, tokens] (got {tuple(path.shape)})")
    B, T = path.shape
    path_p = _ints(path, (B, T), dev, "path")
    counts_p = _ints(counts, (B,), dev, "counts")
    lens_p = _ints(seq_lens, (B,), dev, "seq_lens")
    table_p, ld_table, table_pages = _block_table(block_table, B, dev)
    lens = torch.empty(B, dtype=torch.int32, device=path.device)
    st = lib.hxm_compact_cache(cache, layers, kls, vls, table_p, ld_table, table_pages, lens_p,
                               path_p, counts_p, lens.data_ptr(), B, T, _DT[dtype],
                               _current_stream(dev))
    if st:
        check(st, "hxm_compact_cache")
    return lens


@_on_stream
def copy_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               rows: Optional[torch.Tensor] = None) -> None:
    """Pages copied in all layers' caches (hxm_copy_pages; the caches as
    :func:`compact_cache` takes them), for sequences that fork: page ``dst``[i]
    receives page ``src``[i], or its first ``rows``[i] tokens.  int32 [N] each; -1
    marks padding.  No page may be one pair's dst and another's src or dst."""
    cache, layers, kls, vls, dtype, dev = _kv_layers(k_cache, v_cache)
    N = src.numel()
    src_p, dst_p = _ints(src, (N,), dev, "src"), _ints(dst, (N,), dev, "dst")
    rows_p = None if rows is None else _ints(rows, (N,), dev, "rows")
    st = lib.hxm_copy_pages(cache, layers, kls, vls, src_p, dst_p, rows_p, N, _DT[dtype],
                            _current_stream(dev))
    if st:
        check(st, "hxm_copy_pages")


@_on_stream
def lora_add(y: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
             index: torch.Tensor, scale: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Low-rank adapters of many requests beside a projection they share
    (hxm_lora_add): out[m] = y[m] + scale[a] * (x[m] @ A[a].T) @ B[a].T with
    a = ``index``[m] (int32 [M]; -1: out[m] = y[m]).

    y [M, N] is the projection's output and x [M, K] its input (f16 or bf16);
    A [adapters, R, K] and B [adapters, N, R] contiguous, R a multiple of 8 up
    to 256; scale fp32 [adapters].  ``out`` may be y."""
    dev = _on_current(y, "y")
    _mat(y, "y"), _mat(x, "x")
    dtype = y.dtype
    _dtype(y, _HALVES, "y")
    M, N = y.shape
    K = x.shape[1]
    _tensor(x, dtype, (M, K), dev, "x")
    if A.dim() != 3:
        raise ValueError(f"A must be [adapters, R, {K}] (got {tuple(A.shape)})")
    L, R, _ = A.shape
    _tensor(A, dtype, (L, R, K), dev, "A"), _tensor(B, dtype, (L, N, R), dev, "B")
    if not A.is_contiguous() or not B.is_contiguous():
        raise ValueError("A and B must be contiguous")
    index_p = _ints(index, (M,), dev, "index")
    scale_p = None
    if scale is not None:
        scale = _tensor(scale, torch.float32, (L,), dev, "scale").contiguous()
        scale_p = scale.data_ptr()
    if out is None:
        out = torch.empty_like(y, memory_format=torch.contiguous_format)
    else:
        _out(out, (M, N), (dtype,), y)
    st = lib.hxm_lora_add(y.data_ptr(), _row_ld(y, M, N), x.data_ptr(), _row_ld(x, M, K),
                          A.data_ptr(), B.data_ptr(), L, R, index_p, scale_p, out.data_ptr(),
                          _row_ld(out, M, N), M, N, K, _DT[dtype], _current_stream(dev))
    if st:
        check(st, "hxm_lora_add")
    return out


def tune_gemm(A: torch.Tensor, B_nk: torch.Tensor, out: torch.Tensor, *, reps: int = 5,
              stream=None):
    """Measured tile search on these operands; returns (GemmConfig, report dict).
    reps=0 calibrates the repetitions per config (hxm_calibration_iters of the
    timed warm call against a 10 ms budget, 5 to 1000 launches).  Configs the
    cost model prices out of reach are not launched (``pruned`` in the
    report, with ``model_lb_us`` / ``model_ub_us`` for every config)."""
    import ctypes
    import json
    _mat(A, "A"), _mat(B_nk, "B")
    _dtype(A, (torch.int8, torch.float16, torch.bfloat16), "A")
    if B_nk.dtype != A.dtype:
        raise TypeError(f"A and B must share a dtype (got {A.dtype} and {B_nk.dtype})")
    M, K = A.shape
    N = _b_extent(A, B_nk, "nk")
    _out(out, (M, N), (torch.int32,) if A.dtype == torch.int8 else (A.dtype,), A)
    best = GemmConfig()
    buf = ctypes.create_string_buffer(1 << 16)
    st = lib.hxm_tune_gemm(_code(A), A.data_ptr(), _ld(A), B_nk.data_ptr(), _ld(B_nk),
                           out.data_ptr(), _ld(out), M, N, K, reps, ctypes.byref(best), buf,
                           len(buf), _stream(stream))
    check(st, "hxm_tune_gemm")
    return best, json.loads(buf.value.decode())
