"""Operator-level Python mirror of the reference's kernel interface
(kuiper/source/op/kernels/kernels_interface.h:6-68) over libkuiper_hip.so.

Arguments are torch tensors living on the GPU (torch is only the owner of device memory and
streams here); every call goes through the C-ABI and launches a hand-written HIP kernel on
torch's current stream.  There is no eager/CPU fallback: a CPU tensor is an error.
"""
from __future__ import annotations

import os
from typing import NamedTuple, Optional

import torch

from . import _ffi

ROPE_INTERLEAVED, ROPE_HALF = 0, 1


def _p(t: Optional[torch.Tensor], dtype=None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("kuiperllama_amd.ops: tensors must be on the GPU (no CPU fallback)")
    if not t.is_contiguous():
        raise ValueError("kuiperllama_amd.ops: tensors must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"expected {dtype}, got {t.dtype}")
    return t.data_ptr()


# The handle without building a torch.cuda.Stream for it: 2.5 of the 7.5 us that one
# operator call took on the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


class _Unbound:
    """Stands for csrc/kh_pyops.c, the calls that a decoder layer is made of, until the first of them loads it."""

    def __getattr__(self, name):
        global _n
        import ctypes as C
        import importlib.machinery
        import importlib.util
        from .build import PYOPS_PATH as path
        L = _ffi.lib()
        if not os.path.exists(path):
            raise ImportError(f"{path} is missing: build it with `python -m kuiperllama_amd.build`, which needs this "
                              "interpreter's headers")
        spec = importlib.util.spec_from_loader("kh_pyops", importlib.machinery.ExtensionFileLoader("kh_pyops", path))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.bind(tuple(C.cast(f, C.c_void_p).value for f in (L.kh_add_f32, L.kh_swiglu_f32, L.kh_matmul_f32, L.kh_matmul_q8,
                                                             L.kh_rmsnorm_f32, L.kh_rope_f32, L.kh_mha_f32)),
                 (torch.float32, torch.int32, torch.int8, torch.Tensor, getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
                  _raw_stream, _stream, _ffi.check, C.ArgumentError))
        _n = mod
        return getattr(mod, name)


_n = _Unbound()


def add(in1, in2, out):
    return _n.add(in1, in2, out)


def matmul(x, w, out, scale: float = 1.0):
    return _n.matmul(x, w, out, scale)


def matmul_q8(x, w8, scales, group_size: int, out):
    return _n.matmul_q8(x, w8, scales, group_size, out)


def embedding(tokens, w, out):
    V, dim = w.shape
    _ffi.check(_ffi.lib().kh_embedding_f32(_p(tokens, torch.int32), tokens.numel(),
                                           _p(w, torch.float32), _p(out, torch.float32), dim, V,
                                           _stream()), "kh_embedding_f32")
    return out


def embedding_host_tokens(tokens, w, out):
    """EmbeddingKernel as the reference calls it: `tokens` is a HOST int32 array (numpy); the ids
    travel in the kernel arguments, up to 512 per launch (kh_embedding_f32_host)."""
    import numpy as np
    t = np.ascontiguousarray(tokens, dtype=np.int32)
    _ffi.check(_ffi.lib().kh_embedding_f32_host(t.ctypes.data, t.size, _p(w), _p(out), w.shape[1],
                                                w.shape[0], _stream()), "kh_embedding_f32_host")


def swiglu(a, b, out):
    return _n.swiglu(a, b, out)


def rmsnorm(x, w, out, eps: float):
    return _n.rmsnorm(x, w, out, eps)


def rope(q, k, pos, sin_cache, cos_cache, head_size: int, mode: int):
    """pos: python int, or a 1-element int32 GPU tensor (graph-capturable form)."""
    _n.rope(q, k, pos, sin_cache, cos_cache, head_size, mode)
    return q, k


def sincos_cache(head_size: int, seq_len: int, theta: float, sin_cache, cos_cache):
    _ffi.check(_ffi.lib().kh_sincos_cache_f32(head_size, seq_len, theta,
                                              _p(sin_cache, torch.float32),
                                              _p(cos_cache, torch.float32), _stream()),
               "kh_sincos_cache_f32")
    return sin_cache, cos_cache


def mha(pos, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size, mha_out, q, score,
        kcache, vcache):
    return _n.mha(pos, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size, mha_out, q, score, kcache, vcache)


def mha_prefill(pos0, n_tokens, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size, mha_out, q,
                kcache, vcache):
    """Causal attention of n_tokens consecutive queries (rows of q) on the matrix cores."""
    _ffi.sync_env()  # KH_PG_ATTN_QT
    _ffi.check(_ffi.lib().kh_mha_prefill_f32(
        int(pos0), int(n_tokens), head_num, layer_index, seq_len, kv_dim, kv_mul, head_size,
        _p(mha_out, torch.float32), _p(q, torch.float32), _p(kcache, torch.float32),
        _p(vcache, torch.float32), _stream()), "kh_mha_prefill_f32")
    return mha_out


def mha_decode_workspace(head_num: int, head_size: int, seq_len: int, device):
    """Zeroed workspace tensor for mha_decode (None when no time split is needed)."""
    _ffi.sync_env()  # KH_ATTN_TLONG
    n = int(_ffi.lib().kh_mha_decode_workspace_bytes(head_num, head_size, seq_len))
    if n < 0:
        _ffi.check(n, "kh_mha_decode_workspace_bytes")
    return torch.zeros(n, dtype=torch.uint8, device=device) if n else None


def mha_decode(pos, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size, mha_out, q, kcache,
               vcache, workspace):
    d_pos, ipos = (None, int(pos)) if not torch.is_tensor(pos) else (_p(pos, torch.int32), 0)
    _ffi.check(_ffi.lib().kh_mha_decode_f32(
        d_pos, ipos, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size,
        _p(mha_out, torch.float32), _p(q, torch.float32), _p(kcache, torch.float32),
        _p(vcache, torch.float32), _p(workspace) if workspace is not None else None,
        workspace.numel() if workspace is not None else 0, _stream()), "kh_mha_decode_f32")
    return mha_out


def argmax(logits, out_index):
    _ffi.check(_ffi.lib().kh_argmax_f32(_p(logits, torch.float32), logits.numel(),
                                        _p(out_index, torch.int32), _stream()), "kh_argmax_f32")
    return out_index


def argmax_host(logits) -> int:
    import ctypes as C
    r = C.c_int64(-1)
    _ffi.check(_ffi.lib().kh_argmax_f32_host(_p(logits, torch.float32), logits.numel(),
                                             C.byref(r), _stream()), "kh_argmax_f32_host")
    return int(r.value)


def softmax_(x):
    _ffi.check(_ffi.lib().kh_softmax_f32(_p(x, torch.float32), x.numel(), _stream()),
               "kh_softmax_f32")
    return x


def scale_(scale: float, x):
    _ffi.check(_ffi.lib().kh_scale_f32(scale, _p(x, torch.float32), x.numel(), _stream()),
               "kh_scale_f32")
    return x


def scale_sum(value, scale, out, pos: int, size: int, stride: int):
    _ffi.check(_ffi.lib().kh_scale_sum_f32(_p(value, torch.float32), _p(scale, torch.float32),
                                           _p(out, torch.float32), pos, size, stride, _stream()),
               "kh_scale_sum_f32")
    return out


# ---- many tokens of several sequences ------------------------------------------------------------------------------------
# Tensors of rows are [tokens, heads, elements] in bfloat16 or float32, with any strides of tokens and heads that are multiples
# of 16 bytes and the elements of a head side by side: a slice of a wider row will do.  A cache is two tensors [pages, page_size,
# kv_heads, elements] of that kind.  Query head h goes with key head h // (heads / kv_heads).

_DTYPES = {torch.bfloat16: 1, torch.float32: 2}


class RopeTable(NamedTuple):
    """Angles of one rotation: turns[i] of a 64-bit turn a position for pair i, the factor of rotated pairs."""
    turns: torch.Tensor
    rot_dim: int
    magnitude: float


def rope_turns(rot_dim: int, theta: float, scaling: Optional[dict] = None):
    """(fractions of a turn a position, of 2**64, for each of rot_dim / 2 pairs; factor of rotated pairs).  scaling: as rope_scaling in
    a model's config.json, rope_type "default", "linear", "llama3" or "yarn"."""
    import ctypes as C
    c, kind = None, (scaling or {}).get("rope_type", (scaling or {}).get("type", "default"))
    if kind == "linear":
        c = _ffi.RopeScaling(kind=1, factor=scaling["factor"])
    elif kind == "llama3":
        c = _ffi.RopeScaling(kind=2, factor=scaling["factor"], original=scaling["original_max_position_embeddings"],
                             low=scaling["low_freq_factor"], high=scaling["high_freq_factor"])
    elif kind == "yarn":
        c = _ffi.RopeScaling(kind=3, factor=scaling["factor"], original=scaling["original_max_position_embeddings"],
                             fast=scaling.get("beta_fast", 32.0), slow=scaling.get("beta_slow", 1.0),
                             magnitude=scaling.get("attention_factor") or 0.0)
    elif kind != "default":
        raise ValueError(f"rope_type {kind!r}: default, linear, llama3 or yarn expected")
    turns, magnitude = (C.c_uint64 * max(1, rot_dim // 2))(), C.c_float()
    _ffi.check(_ffi.lib().kh_rope_turns(rot_dim, theta, C.byref(c) if c is not None else None, turns, C.byref(magnitude)), "kh_rope_turns")
    return list(turns)[:rot_dim // 2], magnitude.value


def rope_table(rot_dim: int, theta: float, device, scaling: Optional[dict] = None) -> RopeTable:
    """What rope_tokens and rope_store rotate by (rope_turns), on the device."""
    turns, magnitude = rope_turns(rot_dim, theta, scaling)
    signed = [t - (1 << 64) if t >> 63 else t for t in turns]
    return RopeTable(torch.tensor(signed, dtype=torch.int64, device=device), rot_dim, magnitude)


def _rows(t, dtype, dims, what):
    """Address of rows, their type checked."""
    if not t.is_cuda:
        raise ValueError("kuiperllama_amd.ops: tensors must be on the GPU (no CPU fallback)")
    if t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
    if t.dim() != dims or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{what}: {dims} dimensions with the last one contiguous expected, got {tuple(t.shape)} by {t.stride()}")
    return t.data_ptr()


def _numbers(t, dtype, shape, what):
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {shape} expected, got {tuple(t.shape)}")
    return _p(t, dtype)


def _same_device(*tensors):
    """The one device of the tensors, and its current stream."""
    d = tensors[0].device
    for t in tensors:
        if t.device != d:
            raise ValueError(f"kuiperllama_amd.ops: tensors on {d} and {t.device}")
    return d, torch.cuda.current_stream(d).cuda_stream


def _shape(t, shape, what):
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {shape} expected, got {tuple(t.shape)}")


def _storage_type(t):
    if t.dtype not in _DTYPES:
        raise TypeError(f"expected bfloat16 or float32, got {t.dtype}")
    return _DTYPES[t.dtype]


def _cache(kcache, vcache, dtype, kv_heads):
    c = _ffi.PageCache(k=_rows(kcache, dtype, 4, "kcache"), v=_rows(vcache, dtype, 4, "vcache"))
    if kcache.shape[:3] != vcache.shape[:3] or kcache.shape[2] != kv_heads:
        raise ValueError(f"a cache of {kv_heads} key heads expected, got {tuple(kcache.shape)} and {tuple(vcache.shape)}")
    c.k_page, c.k_slot, c.k_head = kcache.stride()[:3]
    c.v_page, c.v_slot, c.v_head = vcache.stride()[:3]
    c.n_pages, c.page_size = kcache.shape[:2]
    return c


def _rope_rows(q, k, positions, table, mode, q_out, k_out):
    code = _storage_type(q)
    r = _ffi.RopeRows(dtype=code, mode=mode, n_tokens=q.shape[0], head_num=q.shape[1] if q.dim() == 3 else 0, rot_dim=table.rot_dim,
                      magnitude=table.magnitude, turns=_numbers(table.turns, torch.int64, (table.rot_dim // 2,), "table"),
                      positions=_numbers(positions, torch.int32, (q.shape[0],), "positions"))
    r.q, r.k = _rows(q, q.dtype, 3, "q"), _rows(k, q.dtype, 3, "k")
    if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q and k of the same tokens and sizes expected, got {tuple(q.shape)} and {tuple(k.shape)}")
    r.kv_head_num, r.head_size = k.shape[1:]
    r.q_token, r.q_head, r.k_token, r.k_head = *q.stride()[:2], *k.stride()[:2]
    _shape(q_out, tuple(q.shape), "q_out")
    r.q_out = _rows(q_out, q.dtype, 3, "q_out")
    r.qo_token, r.qo_head = q_out.stride()[:2]
    if k_out is not None:
        _shape(k_out, tuple(k.shape), "k_out")
        r.k_out = _rows(k_out, q.dtype, 3, "k_out")
        r.ko_token, r.ko_head = k_out.stride()[:2]
    return r


def rope_tokens(q, k, positions, table: RopeTable, mode: int, q_out=None, k_out=None):
    """Rotates the first table.rot_dim elements of every head of q [tokens, heads, size] and k [tokens, kv_heads, size] by their token's
    position (int32 [tokens]); into q_out and k_out, or in place.  -> (q_out, k_out)"""
    import ctypes as C
    q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
    r = _rope_rows(q, k, positions, table, mode, q_out, k_out)
    d, s = _same_device(q, k, positions, table.turns, q_out, k_out)
    with torch.cuda.device(d):
        _ffi.check(_ffi.lib().kh_rope_tokens(C.byref(r), s), "kh_rope_tokens")
    return q_out, k_out


def rope_store(q, k, v, positions, table: RopeTable, mode: int, kcache, vcache, slots, q_out=None):
    """rope_tokens with the rotated keys, and the values, written into a cache: token t to slot slots[t] % page_size of page
    slots[t] // page_size (int32 [tokens], each its own; negative: not stored).  -> q_out"""
    import ctypes as C
    q_out = q if q_out is None else q_out
    r = _rope_rows(q, k, positions, table, mode, q_out, None)
    c = _cache(kcache, vcache, q.dtype, r.kv_head_num)
    vp = _rows(v, q.dtype, 3, "v")
    _shape(v, (r.n_tokens, r.kv_head_num, vcache.shape[3]), "v")
    if kcache.shape[3] != r.head_size:
        raise ValueError(f"kcache: keys of {r.head_size} expected, got {kcache.shape[3]}")
    sp = _numbers(slots, torch.int32, (r.n_tokens,), "slots")
    d, s = _same_device(q, k, v, positions, table.turns, q_out, kcache, vcache, slots)
    with torch.cuda.device(d):
        _ffi.check(_ffi.lib().kh_rope_store(C.byref(r), vp, v.stride(0), v.stride(1), v.shape[2], C.byref(c), sp, s), "kh_rope_store")
    return q_out


def _attn_rows(q, offsets, out, value_size, kv_heads, scale, window):
    code = _storage_type(q)
    r = _ffi.AttnRows(dtype=code, n_seqs=offsets.numel() - 1, kv_head_num=kv_heads, value_size=value_size, window=window)
    r.q = _rows(q, q.dtype, 3, "q")
    r.n_tokens, r.head_num, r.head_size = q.shape
    r.scale = r.head_size ** -0.5 if scale is None else scale
    r.offsets = _numbers(offsets, torch.int32, (r.n_seqs + 1,), "offsets")
    _shape(out, (r.n_tokens, r.head_num, value_size), "out")
    r.out = _rows(out, q.dtype, 3, "out")
    r.q_token, r.q_head = q.stride()[:2]
    r.o_token, r.o_head = out.stride()[:2]
    return r


def attn_packed(q, k, v, offsets, out, scale: Optional[float] = None, window: int = 0):
    """Causal attention of whole prompts, one behind the other: q [tokens, heads, size], k and v [tokens, kv_heads, size], sequence b
    the tokens offsets[b] .. offsets[b + 1] - 1 (int32).  window > 0: the last `window` keys.  scale: 1 / sqrt(size).  -> out"""
    import ctypes as C
    kp, vp = _rows(k, q.dtype, 3, "k"), _rows(v, q.dtype, 3, "v")
    r = _attn_rows(q, offsets, out, v.shape[2], k.shape[1], scale, window)
    if k.shape[0] != r.n_tokens or k.shape[2] != r.head_size or v.shape[:2] != k.shape[:2]:
        raise ValueError(f"q, k and v of the same tokens expected, got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    d, s = _same_device(q, k, v, offsets, out)
    with torch.cuda.device(d):
        _ffi.check(_ffi.lib().kh_attn_packed(C.byref(r), kp, k.stride(0), k.stride(1), vp, v.stride(0), v.stride(1), s), "kh_attn_packed")
    return out


def attn_paged_workspace(heads: int, kv_heads: int, value_size: int, tokens: int, device):
    """Zeroed workspace of attn_paged for up to `tokens` tokens a call."""
    n = int(_ffi.lib().kh_attn_paged_workspace_bytes(heads, kv_heads, value_size, tokens))
    if n < 0:
        _ffi.check(n, "kh_attn_paged_workspace_bytes")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def attn_paged(q, kcache, vcache, pages, lengths, offsets, out, workspace, scale: Optional[float] = None, window: int = 0,
               max_new: Optional[int] = None):
    """Causal attention of the new tokens of each sequence, q [tokens, heads, size], sequence b the tokens offsets[b] .. offsets[b + 1] - 1,
    over the lengths[b] keys that the pages pages[b] (int32 [sequences, most pages]) of the cache hold of it, the new ones the
    last of them.  window, scale: as attn_packed.  max_new: the most new tokens of a sequence, where the caller knows it (it
    chooses the kernel).  workspace: attn_paged_workspace(...), not shared by calls that may run at the same time.  -> out"""
    import ctypes as C
    r = _attn_rows(q, offsets, out, vcache.shape[-1], kcache.shape[2], scale, window)
    c = _cache(kcache, vcache, q.dtype, r.kv_head_num)
    if kcache.shape[3] != r.head_size:
        raise ValueError(f"kcache: keys of {r.head_size} expected, got {kcache.shape[3]}")
    lp = _numbers(lengths, torch.int32, (r.n_seqs,), "lengths")
    if not pages.is_cuda or pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[0] != r.n_seqs or (pages.stride(1) != 1 and pages.shape[1] > 1):
        raise ValueError("pages: int32 [sequences, pages] on the GPU expected, the pages of a sequence side by side")
    d, s = _same_device(q, kcache, vcache, pages, lengths, offsets, out, workspace)
    with torch.cuda.device(d):
        _ffi.check(_ffi.lib().kh_attn_paged(C.byref(r), C.byref(c), pages.data_ptr(), pages.stride(0), pages.shape[1], lp, max_new or 0,
                                            _p(workspace, torch.uint8), workspace.numel(), s), "kh_attn_paged")
    return out
