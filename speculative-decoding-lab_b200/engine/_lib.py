"""ctypes binding of the sm_100a C-ABI library (``lib/libsdl_b200.so``).

There is no CPU or PyTorch fallback: every entry point below requires the
library and CUDA tensors, and raises when either is missing.  Signatures
mirror ``include/sdl_b200.h``.
"""

from __future__ import annotations

import contextlib
import ctypes
import gc
import os
from typing import Optional

import torch

_PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(_PKG_ROOT, "lib", "libsdl_b200.so")

c_int = ctypes.c_int32
c_i64 = ctypes.c_int64
c_size = ctypes.c_size_t
c_float = ctypes.c_float
c_void = ctypes.c_void_p
c_char_p = ctypes.c_char_p

SDL_F32, SDL_BF16, SDL_F16 = 0, 1, 2

DEVERR_EXHAUSTED = 1
DEVERR_TABLE_OVERFLOW = 2
DEVERR_BAD_INDEX = 4
DEVERR_TIMEOUT = 8
DEVERR_BAD_SLOT = 16
DEVERR_BAD_SAMPLE = 32
DEVERR_UNIFORMS = 64

REL_TRUNCATE = 1
REL_ONLY_IF_LONGER = 2
REL_CLEAR = 4

#: Every symbol ``include/sdl_b200.h`` declares (checked by the CPU test suite).
EXPORTED_SYMBOLS = (
    "sdl_version",
    "sdl_last_error",
    "sdl_block_init",
    "sdl_block_alloc",
    "sdl_block_free",
    "sdl_kv_reserve",
    "sdl_kv_append",
    "sdl_kv_release",
    "sdl_kv_truncate",
    "sdl_spec_commit",
    "sdl_spec_commit_n",
    "sdl_make_kv_tensor_map",
    "sdl_attention_workspace_bytes",
    "sdl_attention_launches",
    "sdl_attention_kernel",
    "sdl_attention_fuses_rope",
    "sdl_paged_attention",
    "sdl_paged_attention_noalloc",
    "sdl_noalloc_scratch_bytes",
    "sdl_paged_decode",
    "sdl_paged_verify",
    "sdl_prefill_chunk",
    "sdl_prefix_attention_workspace_bytes",
    "sdl_prefix_attention_kernel",
    "sdl_prefix_attention",
    "sdl_logits_to_probs",
    "sdl_argmax_rows",
    "sdl_sample_rows",
    "sdl_counter_add",
    "sdl_spec_sample",
    "sdl_spec_sample_scratch_bytes",
    "sdl_sampler_workspace_bytes",
    "sdl_sample_logits_rows",
    "sdl_spec_sample_logits",
    "sdl_spec_sample_logits_n",
    "sdl_set_spec_sampler_mode",
    "sdl_get_error",
    "sdl_rmsnorm",
    "sdl_rope",
    "sdl_silu_mul",
    "sdl_swiglu",
    "sdl_rope_axes",
    "sdl_kv_append_rotary",
)


class SdlKvMeta(ctypes.Structure):
    _fields_ = [
        ("block_table", c_void),
        ("num_blocks", c_void),
        ("seq_lens", c_void),
        ("free_stack", c_void),
        ("free_top", c_void),
        ("is_free", c_void),
        ("err", c_void),
        ("capacity", c_int),
        ("width", c_int),
        ("max_rows", c_int),
        ("block_size", c_int),
    ]


class SdlAttnArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void),
        ("q_sb", c_i64), ("q_sj", c_i64), ("q_sh", c_i64),
        ("out", c_void),
        ("o_sb", c_i64), ("o_sj", c_i64), ("o_sh", c_i64),
        ("out_dtype", c_int),
        ("dtype", c_int),
        ("k_pool", c_void),
        ("v_pool", c_void),
        ("tmap_k", c_void),
        ("tmap_v", c_void),
        ("block_table", c_void), ("width", c_int), ("capacity", c_int),
        ("num_layers", c_int), ("layer", c_int), ("block_size", c_int),
        ("rows", c_void),
        ("k_dense", c_void), ("v_dense", c_void), ("kv_len", c_int),
        ("starts", c_void),
        ("valid_rows", c_void),
        ("B", c_int), ("chunk", c_int), ("Hq", c_int), ("Hkv", c_int), ("head_dim", c_int),
        ("max_limit", c_int),
        ("scale", c_float),
        ("workspace", c_void),
        ("workspace_bytes", c_size),
        ("pages_per_split", c_int),
        ("force_generic", c_int),
        ("kv_heads_per_cta", c_int),
        ("use_umma", c_int),
        ("cluster_merge", c_int),
        ("key_count", c_i64),
        ("mma_layout", c_int),
        ("k_new", c_void),
        ("v_new", c_void),
        ("new_row_stride", c_i64),
        ("err", c_void),
        ("rope_cos", c_void),
        ("rope_sin", c_void),
        ("rope_stride", c_i64),
        ("overlap_layers", c_int),
    ]


class SdlPrefixArgs(ctypes.Structure):
    _fields_ = [
        ("attn", SdlAttnArgs),
        ("table_rows", c_int),
        ("prefix_row", c_int),
        ("prefix_len", c_int),
        ("kernel", c_int),
        ("prefix_split", c_int),
        ("own_split", c_int),
    ]


class SdlRopeArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_void), ("q_row_stride", c_i64),
        ("q_out", c_void), ("q_out_row_stride", c_i64),
        ("k", c_void), ("k_row_stride", c_i64),
        ("k_out", c_void), ("k_out_row_stride", c_i64),
        ("v", c_void), ("v_row_stride", c_i64),
        ("k_pool", c_void), ("v_pool", c_void),
        ("slots", c_void),
        ("table", c_void), ("table_rows", c_i64),
        ("positions", c_void), ("pos_stride", c_i64),
        ("err", c_void),
        ("pos64", c_int),
        ("axes", c_int),
        ("sections", c_int * 4),
        ("num_tokens", c_int), ("Hq", c_int), ("Hkv", c_int), ("head_dim", c_int), ("rotary", c_int),
        ("dtype", c_int),
        ("num_layers", c_int), ("layer", c_int), ("capacity", c_int), ("block_size", c_int),
    ]


_P = ctypes.POINTER
_SIGS = {
    "sdl_version": (c_char_p, []),
    "sdl_last_error": (c_char_p, []),
    "sdl_block_init": (c_int, [c_void, c_void, c_void, c_int, c_void]),
    "sdl_block_alloc": (c_int, [c_void, c_void, c_void, c_int, c_int, c_void, c_void, c_void]),
    "sdl_block_free": (c_int, [c_void, c_void, c_void, c_int, c_int, c_void, c_void, c_void]),
    "sdl_kv_reserve": (c_int, [_P(SdlKvMeta), c_int, c_void, c_void, c_void, c_void, c_void]),
    "sdl_kv_append": (c_int, [c_void, c_void, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_void,
                              c_void, c_void, c_i64, c_void, c_void]),
    "sdl_kv_release": (c_int, [_P(SdlKvMeta), c_int, c_void, c_void, c_void, c_void]),
    "sdl_kv_truncate": (c_int, [_P(SdlKvMeta), c_int, c_void, c_void, c_void]),
    "sdl_spec_commit": (c_int, [_P(SdlKvMeta), _P(SdlKvMeta), c_int, c_void, c_void, c_void, c_int, c_void,
                                c_int, c_void, c_void, c_void, c_void, c_void]),
    "sdl_spec_commit_n": (c_int, [_P(SdlKvMeta), _P(SdlKvMeta), c_int, c_void, c_void, c_void, c_int, c_void,
                                  c_int, c_void, c_void, c_void, c_void, c_void, c_void]),
    "sdl_make_kv_tensor_map": (c_int, [c_void, c_void, c_int, c_i64, c_int, c_int]),
    "sdl_attention_workspace_bytes": (c_size, [_P(SdlAttnArgs)]),
    "sdl_attention_launches": (c_int, [_P(SdlAttnArgs)]),
    "sdl_attention_kernel": (c_int, [_P(SdlAttnArgs)]),
    "sdl_attention_fuses_rope": (c_int, [_P(SdlAttnArgs)]),
    "sdl_paged_attention": (c_int, [_P(SdlAttnArgs), c_void]),
    "sdl_paged_attention_noalloc": (c_int, [_P(SdlAttnArgs), c_void]),
    "sdl_noalloc_scratch_bytes": (c_size, []),
    "sdl_paged_decode": (c_int, [_P(SdlAttnArgs), c_void]),
    "sdl_paged_verify": (c_int, [_P(SdlAttnArgs), c_void]),
    "sdl_prefill_chunk": (c_int, [_P(SdlAttnArgs), c_void]),
    "sdl_prefix_attention_workspace_bytes": (c_size, [_P(SdlPrefixArgs)]),
    "sdl_prefix_attention_kernel": (c_int, [_P(SdlPrefixArgs)]),
    "sdl_prefix_attention": (c_int, [_P(SdlPrefixArgs), c_void]),
    "sdl_logits_to_probs": (c_int, [c_void, c_int, c_i64, c_int, c_int, c_float, c_float, c_int, c_void,
                                    c_i64, c_void]),
    "sdl_argmax_rows": (c_int, [c_void, c_int, c_i64, c_int, c_int, c_void, c_void]),
    "sdl_sample_rows": (c_int, [c_void, c_i64, c_int, c_int, c_void, c_i64, c_void, c_i64, c_void, c_void,
                                c_void]),
    "sdl_counter_add": (c_int, [c_void, c_i64, c_void]),
    "sdl_spec_sample": (c_int, [c_void, c_i64, c_i64, c_void, c_i64, c_i64, c_void, c_void, c_int, c_int,
                                c_int, c_int, c_void, c_i64, c_void, c_i64, c_void, c_void, c_void, c_void,
                                c_void]),
    "sdl_spec_sample_scratch_bytes": (c_size, [c_int]),
    "sdl_sampler_workspace_bytes": (c_size, [c_int, c_int]),
    "sdl_sample_logits_rows": (c_int, [c_void, c_int, c_i64, c_int, c_int, c_float, c_float, c_void, c_i64, c_void,
                                       c_i64, c_void, c_void, c_size, c_void, c_void]),
    "sdl_spec_sample_logits": (c_int, [c_void, c_i64, c_i64, c_void, c_i64, c_i64, c_int, c_float, c_float, c_void,
                                       c_int, c_int, c_int, c_void, c_i64, c_void, c_i64, c_void, c_void, c_void,
                                       c_size, c_void, c_void]),
    "sdl_spec_sample_logits_n": (c_int, [c_void, c_i64, c_i64, c_void, c_i64, c_i64, c_int, c_float, c_float,
                                         c_void, c_int, c_int, c_int, c_void, c_i64, c_void, c_i64, c_void, c_void,
                                         c_void, c_size, c_void, c_void, c_void]),
    "sdl_set_spec_sampler_mode": (c_int, [c_int]),
    "sdl_get_error": (c_int, [c_void, c_void, c_int, c_void]),
    "sdl_rmsnorm": (c_int, [c_void, c_i64, c_void, c_i64, c_void, c_i64, c_void, c_void, c_i64, c_int, c_int, c_float,
                            c_int, c_void]),
    "sdl_rope": (c_int, [c_void, c_i64, c_int, c_int, c_int, c_void, c_i64, c_void, c_i64, c_int, c_void]),
    "sdl_silu_mul": (c_int, [c_void, c_void, c_void, c_i64, c_int, c_void]),
    "sdl_swiglu": (c_int, [c_void, c_i64, c_void, c_i64, c_int, c_int, c_int, c_void]),
    "sdl_rope_axes": (c_int, [_P(SdlRopeArgs), c_void]),
    "sdl_kv_append_rotary": (c_int, [_P(SdlRopeArgs), c_void]),
}

_LIB: Optional[ctypes.CDLL] = None


def load() -> ctypes.CDLL:
    """Load (once) and type the library; raise when it has not been built."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                "sdl_b200 CUDA library missing at {}; build it with "
                "`python speculative-decoding-lab_b200/build_lib.py`".format(LIB_PATH)
            )
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = lib
    return _LIB


def last_error() -> str:
    msg = load().sdl_last_error()
    return msg.decode() if msg else ""


# Entry calls into the library made from this process (each launches one or
# more of its kernels); CUDA-graph replays add the calls their capture made.
_CALLS = [0]


def calls() -> int:
    """Library entry calls so far (``check`` counts every one)."""
    return _CALLS[0]


def count_calls(n: int) -> None:
    """Add ``n`` calls replayed inside a CUDA graph."""
    _CALLS[0] += int(n)


def check(rc: int, what: str) -> None:
    _CALLS[0] += 1
    if rc != 0:
        raise RuntimeError("{} failed (status {}): {}".format(what, rc, last_error()))


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------ shared memory
def _runs(t: torch.Tensor):
    """``t`` as runs of back-to-back elements: the dims over the runs as
    (size, stride) pairs, and a run's length in elements."""
    dims = [(n, st) for n, st in zip(t.shape, t.stride()) if n > 1]
    run = 1
    while dims and dims[-1][1] == run:
        run *= dims.pop()[0]
    return dims, run


def _run_addresses(t: torch.Tensor, dims) -> torch.Tensor:
    at = torch.tensor([t.data_ptr()], dtype=torch.int64, device="cpu")
    for n, st in dims:
        step = torch.arange(n, dtype=torch.int64, device="cpu") * (st * t.element_size())
        at = (at[:, None] + step).reshape(-1)
    return at.sort().values


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements of ``t`` share memory."""
    if t.numel() == 0:
        return False
    dims, run = _runs(t)
    reach = run  # elements that the dims so far span
    for n, st in sorted(dims, key=lambda x: x[1]):
        if st < reach:
            break
        reach += (n - 1) * st
    else:
        return False
    at = _run_addresses(t, dims)
    return bool((at.diff() < run * t.element_size()).any())


def share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of ``a`` and one of ``b`` share memory: by their
    whole spans where those are apart, else run by run."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    lo_a, lo_b = a.data_ptr(), b.data_ptr()
    end_a, end_b = (
        lo + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()
        for lo, t in ((lo_a, a), (lo_b, b)))
    if end_a <= lo_b or end_b <= lo_a:
        return False
    (dims_a, run_a), (dims_b, run_b) = _runs(a), _runs(b)
    at_a, at_b = _run_addresses(a, dims_a), _run_addresses(b, dims_b)
    # the first run of b that ends behind each start in a: does it begin before that run of a ends?
    i = torch.searchsorted(at_b, at_a - run_b * b.element_size(), right=True)
    found = i < at_b.numel()
    return bool((at_b[i[found]] < at_a[found] + run_a * a.element_size()).any())


def same_elements(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``a`` and ``b``, of one shape, are the same elements in place."""
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and all(
        x == y for n, x, y in zip(a.shape, a.stride(), b.stride()) if n > 1)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
# the current device's index, for callers that hold a CUDA tensor (so CUDA is initialised)
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def stream_handle(device: Optional[torch.device] = None) -> int:
    """cudaStream_t of the current stream of ``device`` (as an int)."""
    if _raw_stream is not None and device is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise RuntimeError(
            "{} must be a CUDA tensor: the B200 path has no CPU fallback".format(name)
        )


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return SDL_F32
    if dtype == torch.bfloat16:
        return SDL_BF16
    if dtype == torch.float16:
        return SDL_F16
    raise TypeError("unsupported dtype {} (float32, bfloat16, float16)".format(dtype))


def to_device(values, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Host values -> CUDA tensor without waiting for the stream: built on
    the host and copied with ``non_blocking`` (the copy is queued behind the
    stream's work), where ``torch.tensor(values, device=...)`` would wait for
    every queued kernel first."""
    return torch.tensor(values, dtype=dtype).to(device, non_blocking=True)


def i32(values, device: torch.device) -> torch.Tensor:
    """Host list -> contiguous int32 CUDA tensor (one H2D copy)."""
    if isinstance(values, torch.Tensor):
        return values.to(device=device, dtype=torch.int32).contiguous()
    return torch.tensor(list(values), dtype=torch.int32).to(device, non_blocking=True)


@contextlib.contextmanager
def no_gc():
    """Keep Python's cyclic garbage collector from running inside a CUDA
    graph capture: collecting an unreachable object that holds a captured
    graph would destroy that graph mid-capture and invalidate the capture."""
    was = gc.isenabled()
    gc.disable()
    try:
        yield
    finally:
        if was:
            gc.enable()


class Workspace:
    """Per-device growable fp32 scratch (split-K attention partials under the
    default tag, sampler statistics under ``"sampler"``).

    Buffers start zeroed: a sampler workspace begins with the fused
    sampler's control block, which must be zero before its first use.  A
    buffer that is outgrown is kept alive rather than freed: CUDA graphs
    captured earlier still hold its address.
    """

    _bufs = {}
    _retired = []

    @classmethod
    def get(cls, device: torch.device, nbytes: int, tag: str = "attention") -> torch.Tensor:
        key = (device.type, device.index if device.index is not None else torch.cuda.current_device(), tag)
        buf = cls._bufs.get(key)
        need = max(4, (nbytes + 3) // 4)
        if buf is None or buf.numel() < need:
            if buf is not None:
                cls._retired.append(buf)
            buf = torch.zeros(int(need * 1.25) + 1024, dtype=torch.float32, device=device)
            cls._bufs[key] = buf
        return buf
