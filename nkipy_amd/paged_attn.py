"""Paged flash attention ops on MI355X: NumPy-style signatures over device tensors.

Each op keeps the calling convention of the reference's kernels — positional
arrays in, array out, static options as keywords (README.md:118-152 of the
reference) — with the argument order `(q, k_cache, v_cache, block_tables,
seq_lens, scale) -> out`.  They are hand-kernel ops in the sense of the
reference's `nki_custom_op` (nkipy/src/nkipy/core/nki_op.py:800-884): there is
no CPU implementation behind them, and like that hook on the CPU backend
(nki_op.py:480,557,719-722) they raise NotImplementedError for host arrays.

Ownership follows nkipy/src/nkipy/runtime/device_tensor.py:51-74 and
spike/src/spike/spike_model.py:248-288: the caller may pass `out=` (written in
place, returned); otherwise a new tensor is allocated.  Validation errors are
ValueError (bad shape / dtype / contiguity / device), launch failures are
RuntimeError, mirroring spike_model.py:198-246.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib

F32, BF16, FP8, I8 = 0, 1, 2, 4
_DTYPE_CODE = {torch.float32: F32, torch.bfloat16: BF16, torch.float8_e4m3fn: FP8, torch.int8: I8}

_workspaces = {}
_o_proj_need = {}           # (M, K, N) -> scratch bytes of o_proj's few-rows form (a pure function of the shape)


def _need_device(name, t):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous():
        return                               # the usual case first: these checks run some twenty times per layer call
    if isinstance(t, np.ndarray):
        raise NotImplementedError(
            f"{name} is a NumPy array: the paged attention ops run hand-written HIP kernels and have "
            "no CPU path; pass torch tensors on a ROCm device")
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor on a ROCm device, got {type(t).__name__}")
    if not t.is_cuda:
        raise NotImplementedError(f"{name} lives on {t.device}: the paged attention ops have no CPU path")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _all_on(ref, needed, optional=()):
    """Every (name, tensor) of `needed`, and those of `optional` that are not None, is a contiguous tensor on ref's device:
    `_need_device` and `_same_device` of all of them in one pass, for the calls that a decode loop issues by the thousand."""
    try:
        idx = ref.get_device()
        for _, t in needed:
            if not (t.is_cuda and t.is_contiguous() and t.get_device() == idx):
                break
        else:
            for _, t in optional:
                if t is not None and not (t.is_cuda and t.is_contiguous() and t.get_device() == idx):
                    break
            else:
                return
    except AttributeError:                   # something that is not a tensor: named below
        pass
    named = tuple(needed) + tuple((n, t) for n, t in optional if t is not None)
    for n, t in named:
        _need_device(n, t)
    for n, t in named:
        if t.get_device() != ref.get_device():
            raise ValueError(f"{n} is on {t.device}, expected {ref.device}")


def _check(cond, msg):
    # (the calls a decode loop issues by the thousand spell the raise out where the text is formatted: an argument is
    # formatted whether it is needed or not, and a dozen of them were a quarter of a small call's host time)
    if not cond:
        raise ValueError(msg)


def _same_device(ref, **others):
    idx = ref.get_device()                  # an int: comparing device objects costs several times as much per tensor
    for n, t in others.items():
        if t is not None and t.get_device() != idx:
            raise ValueError(f"{n} is on {t.device}, expected {ref.device}")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device):
    """The current stream of `device` as the C ABI takes it.  torch's raw-stream query when this build has it (a
    fraction of a microsecond; the Stream object of the public call costs several, and a decode step of a small batch
    is bound by the host), the public call otherwise."""
    if _raw_stream is not None and device.index is not None:
        return ctypes.c_void_p(_raw_stream(device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


# (the public calls first make sure that torch's device runtime is up, which a device tensor in hand says already)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_is_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def _on(device):
    """Context in which `device` is the current one for a launch; nothing to switch when it already is
    (the usual case, and the switch costs a few microseconds of a call that launches ten-microsecond kernels)."""
    return _NO_GUARD if _current_device() == device.index else torch.cuda.device(device)


def _ptr(t):
    """A tensor's address as the C signatures take it (a plain int: wrapping it costs as much again)."""
    return t.data_ptr() if t is not None else None


def _raise_on(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc}): {_lib.last_error()}")


def _kv_code(cache, scale_given):
    if cache.dtype == torch.uint8:
        _check(scale_given, "uint8 KV caches are fp8-e4m3fn codes and need k_scale/v_scale")
        return FP8
    if cache.dtype not in _DTYPE_CODE:
        raise ValueError(f"unsupported KV cache dtype {cache.dtype}")
    return _DTYPE_CODE[cache.dtype]


def _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv, what="KV", on_device=False):
    """The scale tables of a pool of codes: one float per (block, kv head) for fp8, per (token, kv head) for int8.
    on_device: the caller has been through `_all_on` with them."""
    shape, text = ((num_blocks, Hkv), "[num_blocks, Hkv]") if kv_code == FP8 else \
                  ((num_blocks, Hkv, block_size), "[num_blocks, Hkv, block_size]")
    if not (k_scale is not None and v_scale is not None):
        raise ValueError(f"{'fp8' if kv_code == FP8 else 'int8'} {what} needs both k_scale and v_scale")
    if on_device and k_scale.shape == shape == v_scale.shape and k_scale.dtype == v_scale.dtype == torch.float32:
        return
    for n, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        _need_device(n, t)
        if t.dtype != torch.float32 or t.shape != shape:
            raise ValueError(f"{n} must be float32 {text}")


def _check_paging(k_cache, v_cache, block_tables, seq_lens, B):
    _check(k_cache.dim() == 4, "k_cache must be [num_blocks, block_size, Hkv, D]")
    _check(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype,
           "v_cache must match k_cache in shape and dtype")
    table = block_tables.shape
    _check(len(table) == 2 and table[0] == B and block_tables.dtype == torch.int32,
           "block_tables must be int32 [B, max_blocks_per_seq]")
    _check(table[1] > 0, "block_tables needs at least one column")
    _check(seq_lens.shape == (B,) and seq_lens.dtype == torch.int32, "seq_lens must be int32 [B]")


def check_block_tables(block_tables, seq_lens, num_blocks, block_size):
    """Debug helper (synchronises): every table entry a sequence uses is a valid block id."""
    bt = block_tables.detach().cpu().numpy()
    sl = seq_lens.detach().cpu().numpy()
    for b in range(bt.shape[0]):
        n = (int(sl[b]) + block_size - 1) // block_size
        _check(n <= bt.shape[1], f"sequence {b}: seq_len {int(sl[b])} needs {n} blocks, table has {bt.shape[1]}")
        used = bt[b, :n]
        _check(used.size == 0 or (used.min() >= 0 and used.max() < num_blocks),
               f"sequence {b}: block table entry outside [0, {num_blocks})")


def _check_variant(sinks, sliding_window, Hq, ref):
    """sinks [Hq] (any float dtype; passed on as float32) and the window size of the gpt-oss attention
    variant (examples/models/gpt_oss/kernels/attention.py:117-148).  Returns (sinks_f32 or None, window int)."""
    win = 0 if sliding_window is None else int(sliding_window)
    _check(win >= 0 and (sliding_window is None or win >= 1), "sliding_window must be None or >= 1")
    win = min(win, 0x7fffffff)      # (the C argument is 32 bits wide: 2^32 + 5 arrived as a window of five keys)
    if sinks is not None:
        _need_device("sinks", sinks)
        _check(sinks.shape == (Hq,), f"sinks must have one logit per q head ([{Hq}])")
        _check(sinks.is_floating_point(), "sinks must be floating point")
        _check(sinks.device == ref.device, f"sinks is on {sinks.device}, expected {ref.device}")
        sinks = sinks.to(torch.float32).contiguous()
    return sinks, win


def decode_workspace_bytes(B, Hq, D, max_seq_len, partition_size) -> int:
    return int(_lib.load().pa_decode_workspace_bytes(B, Hq, D, max_seq_len, partition_size))


_WORKSPACE_SLOTS = 16     # (device, stream) pairs whose eager workspace is kept; the least recently used goes first
_graph_workspaces = {}    # buffers handed out while a stream was being captured: a graph has their address baked in
_graph_retired = []       # ... and those that a later capture outgrew; both are kept until the process ends


def _workspace(device, nbytes, stream=None):
    """Scratch for split-K partials, cached per (device, stream) so that calls on one stream reuse one
    buffer and calls on different streams never share one.

    Eager calls: the cache holds at most _WORKSPACE_SLOTS entries (a server that cycles streams does not
    accumulate device memory); dropping or outgrowing an entry returns its memory to torch's allocator,
    which reuses it in stream order.

    Calls issued while the stream is being captured into a HIP graph take their buffer from a second cache
    that eager calls never touch and that is never evicted or freed: the graph has the address baked in, and
    neither a larger eager call on the same stream after the capture nor the eviction of a stream's entry may
    take that memory away from it.  A capture that needs more than the cached graph buffer retires it (kept
    alive) and takes a new one.  All graphs captured on one capture stream share that one buffer, as all calls
    on a stream do: replays of two of them that overlap on different streams race on it.  Callers that replay
    graphs concurrently pass a `workspace=` of their own per graph, sized with the *_workspace_bytes functions,
    and keep it alive."""
    key = (device, (stream or _stream_ptr(device)).value)
    if (device.type if isinstance(device, torch.device) else torch.device(device).type) == "cuda" and _is_capturing():
        buf = _graph_workspaces.get(key)
        if buf is None or buf.numel() < nbytes:
            if buf is not None:
                _graph_retired.append(buf)
            buf = _graph_workspaces[key] = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
        return buf
    buf = _workspaces.pop(key, None)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    _workspaces[key] = buf              # (re)inserted last: dict order is the LRU order
    while len(_workspaces) > _WORKSPACE_SLOTS:
        _workspaces.pop(next(iter(_workspaces)))
    return buf


class QTransform:
    """Norm and rotation of the Q rows done by the attention kernel as it loads them: the Q half of
    the reference's pre-attention step (QK RMSNorm, examples/models/qwen3/kernels/rmsnorm.py:4-21;
    RoPE at the row's absolute position, rope.py:23-48), bit for bit what `qk_norm_rope_kv_write`
    writes for Q, without that kernel's pass over Q.  rope_cos / rope_sin [max_pos, D/2] bfloat16
    (`rope_tables`); norm_weight [D] bfloat16 or None for rotation only."""

    def __init__(self, rope_cos, rope_sin, norm_weight=None, eps=1e-6):
        self.rope_cos, self.rope_sin, self.norm_weight, self.eps = rope_cos, rope_sin, norm_weight, float(eps)
        self._checked = None                 # (key, struct) of the last validated state

    def _struct(self, D, q):
        # validated once per state: the same object is passed on every call of every step
        key = (D, q.get_device(), q.dtype, id(self.rope_cos), id(self.rope_sin), id(self.norm_weight), self.eps)
        if self._checked is not None and self._checked[0] == key:
            return self._checked[1]
        st = self._build(D, q)
        self._checked = (key, st)
        return st

    def _build(self, D, q):
        for n, t in (("rope_cos", self.rope_cos), ("rope_sin", self.rope_sin)):
            _need_device(n, t)
            _check(t.dim() == 2 and t.shape[1] == D // 2 and t.dtype == torch.bfloat16 and t.shape[0] > 0,
                   f"q_transform.{n} must be bfloat16 [max_pos, D/2]")
        _check(self.rope_sin.shape == self.rope_cos.shape, "q_transform.rope_sin must match rope_cos")
        if self.norm_weight is not None:
            _need_device("norm_weight", self.norm_weight)
            _check(tuple(self.norm_weight.shape) == (D,) and self.norm_weight.dtype == torch.bfloat16,
                   "q_transform.norm_weight must be bfloat16 [D]")
        _check(q.dtype == torch.bfloat16, "q_transform needs bfloat16 q")
        _same_device(q, rope_cos=self.rope_cos, rope_sin=self.rope_sin, norm_weight=self.norm_weight)
        return _lib.QTransformStruct(None if self.norm_weight is None else self.norm_weight.data_ptr(),
                                     self.rope_cos.data_ptr(), self.rope_sin.data_ptr(),
                                     self.rope_cos.shape[0], self.eps)


def q_transform_supported(T, D, block_size) -> bool:
    """Whether the kernel that `decode` (T = 1) or `prefill` picks for bfloat16 q of this shape can
    take a `QTransform`: the matrix-core kernels, which need a power-of-two block size >= 16 and
    head_dim 128 or 64."""
    if block_size < 16 or block_size & (block_size - 1):
        return False
    return D in (64, 128)


def _qt_arg(q_transform, D, q):
    """(struct kept alive by the caller, pointer value or None) for a C call."""
    if q_transform is None:
        return None, None
    _check(isinstance(q_transform, QTransform), "q_transform must be a QTransform")
    st = q_transform._struct(D, q)
    return st, ctypes.addressof(st)


def decode(q, k_cache, v_cache, block_tables, seq_lens, scale, *, k_scale=None, v_scale=None,
           partition_size=512, max_seq_len=None, out=None, workspace=None, validate_tables=False,
           sinks=None, sliding_window=None, q_transform=None):
    """out[b, h] = softmax(q[b, h] . K_b^T * scale) V_b over the paged context.

    q [B, Hq, D] (float32 or bfloat16); k_cache/v_cache [num_blocks, block_size, Hkv, D]
    in q's dtype, or float8_e4m3fn / uint8 codes with k_scale/v_scale [num_blocks, Hkv]
    float32, or int8 codes with k_scale/v_scale [num_blocks, Hkv, block_size] (one scale per token and kv head, as
    `kv_write` leaves them; head_dim 64 or 128, a power-of-two block size >= 16); block_tables int32 [B, max_blocks]; seq_lens int32 [B].
    Over int8 pools a query row goes into the score product as 16-bit integers: elements of at least 2^-6 of the row's
    largest as they are, smaller ones rounded to 2^-15 of it at most; the products with the codes are exact.
    max_seq_len: host-known upper bound of seq_lens (sizes the split-K grid
    without a device sync; default = table capacity).
    sinks [Hq]: per-head logits that join the softmax as one more column and carry no value;
    sliding_window W: only the last W keys are visible (bf16 / fp8 / int8 pools, head_dim 64 or 128).
    q_transform: a `QTransform`; q then holds the rows before norm and rotation (same shapes).
    """
    lib = _lib.load()
    _all_on(q, (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("seq_lens", seq_lens)),
            (("k_scale", k_scale), ("v_scale", v_scale), ("out", out)))
    _check(q.dim() == 3, "q must be [B, Hq, D]")
    B, Hq, D = q.shape
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"unsupported q dtype {q.dtype}")
    _check_paging(k_cache, v_cache, block_tables, seq_lens, B)
    num_blocks, block_size, Hkv, Dk = k_cache.shape
    if Dk != D:
        raise ValueError(f"head_dim mismatch: q has {D}, cache has {Dk}")
    if Hq % Hkv != 0:
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    if D not in (32, 64, 128, 256):
        raise ValueError(f"head_dim {D} not in (32, 64, 128, 256)")
    scaled = k_scale is not None or v_scale is not None
    kv_code = _kv_code(k_cache, scaled)
    q_code = _DTYPE_CODE[q.dtype]
    if kv_code in (FP8, I8):
        if q_code != BF16:
            raise ValueError(f"{'fp8' if kv_code == FP8 else 'int8'} KV needs bfloat16 q")
        _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv, on_device=True)
        if not (kv_code == FP8 or verify_supported(1, D, block_size)):
            raise ValueError(f"int8 KV needs head_dim 64 or 128 and a power-of-two block size >= 16 (D={D}, block_size={block_size})")
    else:
        if kv_code != q_code:
            raise ValueError(f"KV dtype {k_cache.dtype} does not match q dtype {q.dtype}")
        _check(not scaled, "k_scale/v_scale are only valid with an fp8 or int8 KV cache")
    sinks, win = _check_variant(sinks, sliding_window, Hq, q)
    _check(isinstance(partition_size, int) and partition_size > 0, "partition_size must be a positive int")
    cap = block_tables.shape[1] * block_size
    msl = cap if max_seq_len is None else int(max_seq_len)
    if not (0 < msl <= cap):
        raise ValueError(f"max_seq_len {msl} outside (0, {cap}]")
    if validate_tables:
        check_block_tables(block_tables, seq_lens, num_blocks, block_size)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out.shape == q.shape and out.dtype == q.dtype, "out must match q in shape and dtype")
    qt_keep, qt_ptr = _qt_arg(q_transform, D, q)
    with _on(q.device):
        need = int(lib.pa_decode_workspace_bytes_for(B, Hq, Hkv, D, block_size, msl, partition_size, q_code, kv_code))
        stream = _stream_ptr(q.device)
        if workspace is None:
            workspace = _workspace(q.device, need, stream) if need else None
        else:
            _need_device("workspace", workspace)
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace needs {need} bytes")
        ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
        rc = lib.pa_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                           _ptr(block_tables), _ptr(seq_lens), _ptr(out), _ptr(workspace), ws_bytes,
                           B, Hq, Hkv, D, block_size, block_tables.shape[1], num_blocks, msl,
                           float(scale), partition_size, q_code, kv_code, _ptr(sinks), win, qt_ptr, stream)
    _raise_on(rc, "pa_decode")
    return out


# prefill() takes the verify kernel up to this many (query token, q head) rows per kv head: the measured
# crossover against the tiled kernel (rows packed over the kv group, key tiles split over workgroups when
# the grid is small) lies between 16 and 48 rows for batches of 1 to 64 sequences
VERIFY_MAX_ROWS = 32
VERIFY_MAX_ROWS_FP8 = 256     # fp8 pools: the tiled kernel has no packed-rows form for them (B = 64, 4 K prefix: T = 64 718 vs 810 us)
# bf16 pools of head dim 128, more than 16 rows per kv head.  Up to VERIFY_MAX_ROWS rows the verify kernel gives a kv
# head two 16-row waves, each of which streams every tile, and from this many (sequence x bound) tokens on the tiled
# kernel's packed rows are ahead (32 / 8 heads, T = 8, ragged contexts up to the bound, us verify / tiled: B = 8 behind
# 2 K 22.9 / 23.5, behind 4 K 41.0 / 31.3; B = 16 behind 1 K 20.2 / 22.6, behind 2 K 43.0 / 30.1; B = 32 behind 1 K 35.8 /
# 29.5; B = 64 behind 2 K 90.3 / 72.0).  Beyond VERIFY_MAX_ROWS a small call -- few sequences, a bound of a few thousand
# tokens -- is still faster on the verify kernel's fixed partitions (T = 16, us verify / tiled: B = 1 behind 1 K 14.1 /
# 21.0, behind 4 K 20.9 / 25.1; B = 2 behind 2 K 19.7 / 22.4; B = 4 behind 500 15.9 / 18.9), up to this many
# (sequence x row x bound) products.
TILED_FROM_TOKENS = 20_000
VERIFY_SMALL_CALL = 300_000


def prefill_route(B, T, Hq, Hkv, D, block_size, fp8=False, window=0, bound=None) -> str:
    """Which kernel `prefill` takes for a shape: "verify" (the decode-shaped kernel) or "tiled".  bound: what the
    caller knows of the longest context (None: nothing)."""
    can_verify = verify_supported(T, D, block_size)
    # the tiled kernel is built for bf16 pools and head_dim 128; what it cannot take goes to the verify kernel
    rows = T * (Hq // Hkv)
    if D == 64:
        # the tiled kernel takes head dim 64 two kv heads at a time (not a single kv head); below 384 rows per kv head, and for small
        # batches, the verify kernel is faster (measured crossover, as in pa_prefill itself: 64 / 8 heads, us verify /
        # tiled, T = 40: B = 8 behind 1 K 30.5 / 39.9, behind 4 K 58.0 / 74.6; T = 48: B = 8 behind 2 K 48.2 / 45.1)
        return "tiled" if not can_verify or (Hkv >= 2 and B >= 8 and rows >= 384) else "verify"
    if not can_verify:
        return "tiled"
    if D != 128:
        return "verify"
    if fp8:
        return "verify" if window > 0 or rows <= VERIFY_MAX_ROWS_FP8 else "tiled"
    if rows <= 16 or (window > 0 and rows <= VERIFY_MAX_ROWS):
        return "verify"
    if rows <= VERIFY_MAX_ROWS:
        if bound is None:
            return "tiled" if B >= 16 else "verify"
        return "tiled" if B >= 8 and B * bound >= TILED_FROM_TOKENS else "verify"
    return "verify" if bound is not None and window == 0 and B * rows * bound <= VERIFY_SMALL_CALL else "tiled"


def verify_supported(T, D, block_size) -> bool:
    """Shapes the verify kernel is built for."""
    return T <= 64 and D in (64, 128) and block_size >= 16 and block_size & (block_size - 1) == 0


def prefill(q, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, *, k_scale=None, v_scale=None,
            out=None, workspace=None, route=None, validate_tables=False, sinks=None, sliding_window=None,
            q_transform=None, max_seq_len=None):
    """Chunked prefill against a cached prefix (causal).

    q [B, T, Hq, D] bfloat16 holds the last query_lens[b] tokens of each sequence
    (rows t >= query_lens[b] are padding; their output is zero); token i sees keys
    j <= seq_lens[b] - query_lens[b] + i of the paged context, which already
    contains the new tokens' K/V.

    Two kernels stand behind it.  Short query runs -- speculative verify: up to 16 (token, q head) rows per
    kv head always, up to VERIFY_MAX_ROWS for small batches and short bounds, more for a handful of sequences
    under a bound of a few thousand tokens (`prefill_route`) -- go through the decode kernel with the
    (token, head) pairs as its query rows
    (HBM-bound: the context is read once per kv head); everything else through the tiled
    matrix-core prefill kernel (head_dim 128, and 64 with two or more kv heads; long query runs
    at head_dim 64 over a single kv head go through the verify kernel 64 tokens at a time).
    `route` = "verify" or "tiled" forces one.  fp8 pools
    (float8_e4m3fn / uint8 codes with k_scale, v_scale) work on both; int8 pools on the verify kernel only (longer runs:
    `read_kv` and `packed_prefill`).  sinks and sliding_window are
    as in `decode`, the window counted back from each query token; so is q_transform, the position of
    row t being seq_lens[b] - query_lens[b] + t.
    max_seq_len: host-known upper bound of seq_lens, as in `decode`; with it a small verify call (a few
    short sequences, or a short sliding window) takes fixed partitions instead of the balanced schedule, whose
    fixed cost dominates at that size.  For the tiled kernel it is a hint: a chunk with less than twice its own
    length cached in front of it (max_seq_len < 3 T) runs unsplit, which is faster there.
    """
    lib = _lib.load()
    _all_on(q, (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("seq_lens", seq_lens),
                ("query_lens", query_lens)), (("k_scale", k_scale), ("v_scale", v_scale), ("out", out)))
    _check(q.dim() == 4, "q must be [B, T, Hq, D]")
    B, T, Hq, D = q.shape
    _check(q.dtype == torch.bfloat16, "prefill supports bfloat16 only")
    _check_paging(k_cache, v_cache, block_tables, seq_lens, B)
    scaled = k_scale is not None or v_scale is not None
    kv_code = _kv_code(k_cache, scaled)
    _check(kv_code in (BF16, FP8, I8), "prefill needs a bfloat16, fp8 or int8 KV cache")
    _check(query_lens.shape == (B,) and query_lens.dtype == torch.int32, "query_lens must be int32 [B]")
    num_blocks, block_size, Hkv, Dk = k_cache.shape
    if Dk != D:
        raise ValueError(f"head_dim mismatch: q has {D}, cache has {Dk}")
    if Hq % Hkv != 0:
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    if kv_code in (FP8, I8):
        _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv, on_device=True)
    else:
        _check(not scaled, "k_scale/v_scale are only valid with an fp8 or int8 KV cache")
    _check(route in (None, "verify", "tiled"), "route must be None, 'verify' or 'tiled'")
    sinks, win = _check_variant(sinks, sliding_window, Hq, q)
    can_verify = verify_supported(T, D, block_size)
    if kv_code == I8:
        # only the decode-shaped kernel reads int8 pools: long query runs read the pool back (read_kv) for packed_prefill
        if not (route != "tiled" and can_verify):
            raise ValueError(f"prefill over an int8 pool takes runs of up to 64 tokens (the verify kernel: head_dim 64 or 128, a power-of-two "
                             f"block size >= 16; T={T}, D={D}, block_size={block_size}); longer ones go through read_kv and packed_prefill")
        route = "verify"
    if route is None:
        route = prefill_route(B, T, Hq, Hkv, D, block_size, kv_code == FP8, win,
                              None if max_seq_len is None else int(max_seq_len))
    if route == "verify":
        if not (can_verify):
            raise ValueError(f"the verify kernel needs T <= 64, head_dim 64 or 128 and a power-of-two block size >= 16 "
                             f"(T={T}, D={D}, block_size={block_size})")
    if validate_tables:
        check_block_tables(block_tables, seq_lens, num_blocks, block_size)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out.shape == q.shape and out.dtype == q.dtype, "out must match q in shape and dtype")
    qt_keep, qt_ptr = _qt_arg(q_transform, D, q)
    stream = _stream_ptr(q.device)
    cap = block_tables.shape[1] * block_size
    msl = 0 if max_seq_len is None else int(max_seq_len)
    if not (max_seq_len is None or 0 < msl <= cap):
        raise ValueError(f"max_seq_len {msl} outside (0, {cap}]")
    if route == "verify":
        need = int(lib.pa_verify_workspace_bytes(B, T, Hq, D))
        if workspace is None:
            workspace = _workspace(q.device, need, stream)
        else:
            _need_device("workspace", workspace)
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace needs {need} bytes")
        ws_bytes = workspace.numel() * workspace.element_size()
        with _on(q.device):
            rc = lib.pa_verify(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                               _ptr(block_tables), _ptr(seq_lens), _ptr(query_lens), _ptr(out),
                               _ptr(workspace), ws_bytes, B, T, Hq, Hkv, D, block_size,
                               block_tables.shape[1], num_blocks, msl, float(scale), kv_code, _ptr(sinks), win,
                               qt_ptr, stream)
        _raise_on(rc, "pa_verify")
        return out
    with _on(q.device):
        need = int(lib.pa_prefill_workspace_bytes(B, T, Hq, Hkv, D, block_size, block_tables.shape[1]))
        if workspace is None:
            workspace = _workspace(q.device, need, stream) if need else None
        else:
            _need_device("workspace", workspace)
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace needs {need} bytes")
        ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
        rc = lib.pa_prefill(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                            _ptr(block_tables), _ptr(seq_lens),
                            _ptr(query_lens), _ptr(out), B, T, Hq, Hkv, D, block_size,
                            block_tables.shape[1], num_blocks, msl, float(scale), BF16, kv_code, _ptr(sinks), win,
                            _ptr(workspace), ws_bytes, qt_ptr, stream)
    _raise_on(rc, "pa_prefill")
    return out


def verify(q, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, **kw):
    """Speculative verify (gpt_oss/kernels/attention.py:80-100 with seq_len = K+1): prefill through
    the decode-shaped kernel whatever T * (Hq / Hkv) is."""
    return prefill(q, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, route="verify", **kw)


def blocksparse_prefill(q, k, v, scale, *, block=64, local_blocks=4, vert_stride=8, out=None):
    """Block-sparse causal prefill over dense q [B, S, Hq, D], k/v [B, S, Hkv, D] (bfloat16).

    q block i attends k block j iff j <= i and (i - j < local_blocks or
    (j + h % vert_stride) % vert_stride == 0); token-causal inside a block.
    """
    lib = _lib.load()
    for n, t in (("q", q), ("k", k), ("v", v)):
        _need_device(n, t)
    _check(q.dim() == 4 and k.dim() == 4, "q must be [B, S, Hq, D], k/v [B, S, Hkv, D]")
    B, S, Hq, D = q.shape
    _check(q.dtype == torch.bfloat16 and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16,
           "blocksparse_prefill supports bfloat16 only")
    _check(v.shape == k.shape and k.shape[0] == B and k.shape[1] == S and k.shape[3] == D,
           "k/v must be [B, S, Hkv, D] matching q")
    Hkv = k.shape[2]
    _check(Hq % Hkv == 0, f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    _check(block == 64, "sparsity block must be 64")
    _check(local_blocks >= 1 and vert_stride >= 1, "local_blocks and vert_stride must be >= 1")
    _same_device(q, k=k, v=v, out=out)
    if out is None:
        out = torch.empty_like(q)
    else:
        _need_device("out", out)
        _check(out.shape == q.shape and out.dtype == q.dtype, "out must match q in shape and dtype")
    with _on(q.device):
        rc = lib.pa_blocksparse_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, S, Hq, Hkv, D, block,
                                        int(local_blocks), int(vert_stride), float(scale), BF16,
                                        _stream_ptr(q.device))
    _raise_on(rc, "pa_blocksparse_prefill")
    return out


_packed_need = {}           # shape key -> scratch bytes of packed_prefill (a pure function of the shape)


def packed_prefill(q, k, v, cu_seqlens, scale, *, cu_seqlens_k=None, query_lens=None, seq_lens=None, max_seq_len=None,
                   sinks=None, sliding_window=None, out=None, workspace=None):
    """Causal attention over whole prompts of different lengths, packed row behind row, with dense K and V.

    q [Nq, Hq, D], k / v [Nk, Hkv, D] bfloat16 (head_dim 64 or 128); sequence i owns rows cu_seqlens[i] ..
    cu_seqlens[i + 1] - 1 of q and of the result, and rows cu_seqlens_k[i] .. of k and v (default: the same rows).
    The attention of examples/models/qwen3/kernels/attention.py:112-144 for each sequence; with more keys than queries
    the queries are the last ones (gpt_oss/kernels/attention.py:85,127-135): query t of n sees keys j <= c - n + t of c.
    This is the prompt's own attention, before or beside the cache write (`kv_write` with the same cu_seqlens), and,
    with keys that `read_kv` has read back, that of the next chunk of a prompt whose first part is cached.

    q, k and v may be slices of a wider tensor (the heads of a token adjacent, any token stride that is a multiple of 8
    elements): the output of a fused projection as it is.  cu_seqlens int32 [num_seqs + 1].
    query_lens / seq_lens int32 [num_seqs]: of a sequence's rows only the first query_lens[i] are queries and the first
    seq_lens[i] keys (rows laid out with room to spare); the other query rows are padding, zero in the result, and the
    other keys are never read.  A query that sees no key gets zeros; rows that belong to no sequence are left as they
    are (whatever the memory held in a result allocated here).
    An infinity or a NaN in a row reaches the queries that see it (a V row's in its own columns) and no others; the rows
    whose tiles it spoilt are computed again, which costs such calls up to twice the time and more.
    max_seq_len: host-known upper bound of a sequence's keys; sizes the split of calls with few queries over many keys
    (default: Nk where that is at least three times Nq, else twice the mean of the sequences' keys).  sinks [Hq] /
    sliding_window as in `decode`, the window counted back from each query.
    """
    lib = _lib.load()
    qs, ks, vs = _token_rows("q", q), _token_rows("k", k), _token_rows("v", v)
    Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[:2]
    _check(k.shape[2] == D and v.shape == k.shape, "k and v must be [Nk, Hkv, D] with q's D")
    if not (Hkv > 0 and Hq > 0 and Hq % Hkv == 0):
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} must be 64 or 128")
    _all_on(q, (("cu_seqlens", cu_seqlens),), (("cu_seqlens_k", cu_seqlens_k), ("query_lens", query_lens), ("seq_lens", seq_lens), ("out", out)))
    _same_device(q, k=k, v=v)
    _check(cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1, "cu_seqlens must be int32 [num_seqs + 1]")
    S = cu_seqlens.shape[0] - 1
    _check_cu("cu_seqlens", cu_seqlens, S)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens
        if Nk != Nq:
            raise ValueError(f"k has {Nk} rows, q {Nq}: give cu_seqlens_k")
    else:
        _check_cu("cu_seqlens_k", cu_seqlens_k, S)
    for n, t in (("query_lens", query_lens), ("seq_lens", seq_lens)):
        if t is not None:
            if not (t.shape == (S,) and t.dtype == torch.int32):
                raise ValueError(f"{n} must be int32 [num_seqs]")
    if not (max_seq_len is None or int(max_seq_len) > 0):
        raise ValueError(f"max_seq_len {max_seq_len} must be positive")
    bound = 0 if max_seq_len is None else min(int(max_seq_len), Nk)
    sinks, win = _check_variant(sinks, sliding_window, Hq, q)
    if out is None:
        out = torch.empty((Nq, Hq, D), dtype=torch.bfloat16, device=q.device)
    else:
        _need_device("out", out)
        if not (tuple(out.shape) == (Nq, Hq, D) and out.dtype == torch.bfloat16):
            raise ValueError(f"out must be bfloat16 {(Nq, Hq, D)}")
    with _on(q.device):
        stream = _stream_ptr(q.device)
        key = (S, Nq, Nk, Hq, Hkv, D, bound, win)
        need = _packed_need.get(key)
        if need is None:
            if len(_packed_need) >= 4096:
                _packed_need.clear()
            need = _packed_need[key] = int(lib.pa_packed_prefill_workspace_bytes_for(*key))
        if workspace is None:
            workspace = _workspace(q.device, need, stream) if need else None
        else:
            _need_device("workspace", workspace)
            _same_device(q, workspace=workspace)
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace needs {need} bytes")
        ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
        rc = lib.pa_packed_prefill(_ptr(q), _ptr(k), _ptr(v), qs, ks, vs, _ptr(cu_seqlens), _ptr(cu_seqlens_k), _ptr(query_lens),
                                   _ptr(seq_lens), _ptr(out), _ptr(workspace), ws_bytes, S, Nq, Nk, Hq, Hkv, D, bound,
                                   float(scale), BF16, _ptr(sinks), win, stream)
    _raise_on(rc, "pa_packed_prefill")
    return out


def packed_prefill_workspace_bytes(num_seqs: int, total_q: int, total_k: int, Hq: int, Hkv: int, D: int, max_seq_len: int,
                                   sliding_window=None) -> int:
    """Scratch bytes `packed_prefill` would use (0 for calls that take none); max_seq_len 0: the call gives none."""
    return int(_lib.load().pa_packed_prefill_workspace_bytes_for(num_seqs, total_q, total_k, Hq, Hkv, D, max_seq_len,
                                                                 min(sliding_window or 0, 0x7fffffff)))


def gather_kv(cache, block_tables, seq_lens, max_seq_len=None):
    """Materialise the block-table gather: [B, max_seq_len, Hkv, D], zero past seq_lens[b]."""
    lib = _lib.load()
    for n, t in (("cache", cache), ("block_tables", block_tables), ("seq_lens", seq_lens)):
        _need_device(n, t)
    _check(cache.dim() == 4, "cache must be [num_blocks, block_size, Hkv, D]")
    B = block_tables.shape[0]
    _check(block_tables.dim() == 2 and block_tables.dtype == torch.int32, "block_tables must be int32 [B, max_blocks]")
    _check(seq_lens.shape == (B,) and seq_lens.dtype == torch.int32, "seq_lens must be int32 [B]")
    num_blocks, block_size, Hkv, D = cache.shape
    cap = block_tables.shape[1] * block_size
    msl = cap if max_seq_len is None else int(max_seq_len)
    if not (0 <= msl <= cap):
        raise ValueError(f"max_seq_len {msl} outside [0, {cap}]")
    out = torch.empty((B, msl, Hkv, D), dtype=cache.dtype, device=cache.device)
    with _on(cache.device):
        rc = lib.pa_gather_kv(_ptr(cache), _ptr(block_tables), _ptr(seq_lens), _ptr(out), B, Hkv, D,
                              block_size, block_tables.shape[1], num_blocks, msl, cache.element_size(),
                              _stream_ptr(cache.device))
    _raise_on(rc, "pa_gather_kv")
    return out


def _token_rows(name, t, dtype=torch.bfloat16):
    """Packed rows [tokens, heads, D] on the device whose tokens may lie apart (a slice of a wider projection output): the
    heads and their elements are adjacent, and the token stride is a multiple of 8 elements.  Returns the token stride."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _need_device(name, t)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, D]")
    n, heads, D = t.shape
    row = heads * D
    if t.is_contiguous():
        step = row
    else:
        step, across, along = t.stride()
        if (along != 1 and D != 1) or (across != D and heads != 1):
            raise ValueError(f"{name}: the heads of a token must be adjacent rows of D elements (strides {t.stride()})")
        if n <= 1:
            step = row
        elif step % 8 != 0 or step < row:
            raise ValueError(f"{name}: the token stride {step} must be a multiple of 8 elements and at least a token's row")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.data_ptr() % 16 != 0:
        raise ValueError(f"{name} must start on a 16-byte boundary")
    return step


def _check_cu(name, cu, n):
    _need_device(name, cu)
    if not (cu.dim() == 1 and cu.dtype == torch.int32 and cu.shape[0] == n + 1):
        raise ValueError(f"{name} must be int32 [{n + 1}]: where each sequence's rows begin")


def kv_write(k_new, v_new, k_cache, v_cache, block_tables, seq_lens, query_lens, *, k_scale=None, v_scale=None, cu_seqlens=None):
    """Write the new tokens' K/V into the paged pool, in place, before the attention call.

    The reference's `cache_k[:, query_pos] = xk` with query_pos = start_pos + arange(seq_len)
    (examples/models/gpt_oss/kernels/attention.py:85,92-100): token t < query_lens[b] of sequence
    b lands at position seq_lens[b] - query_lens[b] + t, i.e. in pool row
    (block_tables[b, pos // block_size], pos % block_size).  k_new/v_new [B, T, Hkv, D] are
    bfloat16 (float32 for a float32 pool).  float8_e4m3fn pools are quantised on the way in and
    k_scale/v_scale [num_blocks, Hkv] float32 are maintained (running absmax / 448 per block and
    kv head; earlier rows of a block are re-encoded when its scale grows).  int8 pools take codes
    round(x / s) (nearest even) with s = absmax / 127 of the token's row of a kv head (1 for a row of
    zeros), kept in k_scale/v_scale [num_blocks, Hkv, block_size] float32: a row's scale is its own, so
    a written row never changes again (head_dim 32, 64, 128 or 256).  A row that holds an infinity or a NaN
    gets the scale NaN: it reads back as NaN.

    cu_seqlens int32 [B + 1]: the new rows come packed, k_new/v_new [tokens, Hkv, D] bfloat16 with token t of
    sequence b in row cu_seqlens[b] + t (bfloat16 and int8 pools); a query length beyond the cu_seqlens[b + 1] -
    cu_seqlens[b] rows of a sequence counts as their number, and the rows may be slices of a wider tensor (any token stride that is a
    multiple of 8 elements).

    Returns None: the pool tensors are the outputs, aliased to the inputs as the reference's cache tensors are
    (examples/models/qwen3/qwen3.py:289-301).
    """
    lib = _lib.load()
    packed = cu_seqlens is not None
    _all_on(k_cache, (("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("seq_lens", seq_lens),
                      ("query_lens", query_lens)) + (() if packed else (("k_new", k_new), ("v_new", v_new))),
            (("k_scale", k_scale), ("v_scale", v_scale), ("cu_seqlens", cu_seqlens)))
    _check(k_cache.dim() == 4, "k_cache must be [num_blocks, block_size, Hkv, D]")
    _check(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype, "v_cache must match k_cache")
    if k_cache.dtype not in _DTYPE_CODE:
        raise ValueError(f"unsupported pool dtype {k_cache.dtype}")
    kv_dtype = _DTYPE_CODE[k_cache.dtype]
    _check(block_tables.dim() == 2 and block_tables.dtype == torch.int32, "block_tables must be int32 [B, max_blocks]")
    if packed:
        if kv_dtype not in (BF16, I8):
            raise ValueError(f"packed rows go into bfloat16 or int8 pools (a float8 pool's scales belong to whole blocks), got {k_cache.dtype}")
        strides = _token_rows("k_new", k_new), _token_rows("v_new", v_new)
        B = block_tables.shape[0]
        _check_cu("cu_seqlens", cu_seqlens, B)
        Hkv, D = k_new.shape[1:]
    else:
        _check(k_new.dim() == 4, "k_new must be [B, T, Hkv, D]")
        B, T, Hkv, D = k_new.shape
        want = torch.float32 if kv_dtype == F32 else torch.bfloat16
        if k_new.dtype != want:
            raise ValueError(f"k_new must be {want} for a {k_cache.dtype} pool, got {k_new.dtype}")
    _check(v_new.shape == k_new.shape and v_new.dtype == k_new.dtype, "v_new must match k_new")
    num_blocks, block_size = k_cache.shape[:2]
    if tuple(k_cache.shape[2:]) != (Hkv, D):
        raise ValueError(f"pool rows are {tuple(k_cache.shape[2:])}, new rows {(Hkv, D)}")
    _check(block_tables.shape[0] == B, "block_tables must be int32 [B, max_blocks]")
    _check(seq_lens.shape == (B,) and seq_lens.dtype == torch.int32, "seq_lens must be int32 [B]")
    _check(query_lens.shape == (B,) and query_lens.dtype == torch.int32, "query_lens must be int32 [B]")
    if kv_dtype in (FP8, I8):
        _check_scales(kv_dtype, k_scale, v_scale, num_blocks, block_size, Hkv, "pool", True)
    else:
        _check(k_scale is None and v_scale is None, "k_scale / v_scale are for float8 and int8 pools only")
    if not (kv_dtype != I8 and not packed or D in (32, 64, 128, 256)):
        raise ValueError(f"int8 pools and packed rows need head_dim 32, 64, 128 or 256 (got {D})")
    if packed:
        _same_device(k_cache, k_new=k_new, v_new=v_new)
    with _on(k_new.device):
        if packed:
            rc = lib.pa_kv_write_packed(_ptr(k_new), _ptr(v_new), *strides, _ptr(cu_seqlens), k_new.shape[0], _ptr(k_cache),
                                        _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(block_tables), _ptr(seq_lens),
                                        _ptr(query_lens), B, Hkv, D, block_size, block_tables.shape[1], num_blocks, kv_dtype,
                                        _stream_ptr(k_new.device))
        else:
            rc = lib.pa_kv_write(_ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache),
                                 _ptr(k_scale) if k_scale is not None else None,
                                 _ptr(v_scale) if v_scale is not None else None,
                                 _ptr(block_tables), _ptr(seq_lens), _ptr(query_lens),
                                 B, T, Hkv, D, block_size, block_tables.shape[1], num_blocks, kv_dtype,
                                 _stream_ptr(k_new.device))
    _raise_on(rc, "pa_kv_write")


def read_kv(k_cache, v_cache, block_tables, seq_lens, cu_seqlens, total_tokens=None, *, k_scale=None, v_scale=None, out=None):
    """Read a paged cache back as dense bfloat16 rows: token t < seq_lens[b] of sequence b becomes row cu_seqlens[b] + t of
    the results (k, v), [total_tokens, Hkv, D] each -- what `packed_prefill` takes as keys and values of a chunk whose
    first part is cached.

    The block-table gather (np.take of the pool, nkipy/src/nkipy/core/tensor.py:575-640) with the pool's codes
    multiplied by their scales: int8 pools with k_scale/v_scale [num_blocks, Hkv, block_size], float8_e4m3fn / uint8
    codes with [num_blocks, Hkv]; bfloat16 pools come out bit for bit.  cu_seqlens int32 [B + 1]; a sequence gets
    at most cu_seqlens[b + 1] - cu_seqlens[b] rows.  total_tokens: rows of the results, known on the host (at least
    cu_seqlens[B] for every row to have its place).  out: the pair (k, v) to write into (then total_tokens may be left
    out); rows on which no token falls are left as they are -- with results allocated here they hold whatever the
    memory held.
    """
    lib = _lib.load()
    out0, out1 = (None, None) if not isinstance(out, (tuple, list)) or len(out) != 2 else out
    _all_on(k_cache, (("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("seq_lens", seq_lens),
                      ("cu_seqlens", cu_seqlens)), (("k_scale", k_scale), ("v_scale", v_scale), ("out[0]", out0), ("out[1]", out1)))
    _check(block_tables.dim() == 2, "block_tables must be int32 [B, max_blocks_per_seq]")
    B = block_tables.shape[0]
    _check_paging(k_cache, v_cache, block_tables, seq_lens, B)
    num_blocks, block_size, Hkv, D = k_cache.shape
    scaled = k_scale is not None or v_scale is not None
    kv_code = _kv_code(k_cache, scaled)
    _check(kv_code != F32, "read_kv takes bfloat16, float8_e4m3fn / uint8 and int8 pools")
    if kv_code in (FP8, I8):
        _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv, "pool", True)
    else:
        _check(not scaled, "k_scale / v_scale are for float8 and int8 pools only")
    if D % 8 != 0:
        raise ValueError(f"head_dim {D} must be a multiple of 8")
    _check_cu("cu_seqlens", cu_seqlens, B)
    if out is None:
        _check(total_tokens is not None, "total_tokens (rows of the results) is needed without out")
        N = int(total_tokens)
        if N < 0:
            raise ValueError(f"total_tokens {N} is negative")
        out0 = torch.empty((N, Hkv, D), dtype=torch.bfloat16, device=k_cache.device)
        out1 = torch.empty_like(out0)
    else:
        _check(out0 is not None and out1 is not None, "out must be the pair (k, v)")
        for n, t in (("out[0]", out0), ("out[1]", out1)):
            if not (t.dim() == 3 and tuple(t.shape[1:]) == (Hkv, D) and t.dtype == torch.bfloat16 and t.shape[0] == out0.shape[0]):
                raise ValueError(f"{n} must be bfloat16 [tokens, {Hkv}, {D}]")
        N = out0.shape[0]
        if not (total_tokens is None or int(total_tokens) == N):
            raise ValueError(f"out has {N} rows, total_tokens says {total_tokens}")
    with _on(k_cache.device):
        rc = lib.pa_read_kv(_ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(block_tables), _ptr(seq_lens),
                            _ptr(cu_seqlens), _ptr(out0), _ptr(out1), N, B, Hkv, D, block_size, block_tables.shape[1],
                            num_blocks, kv_code, _stream_ptr(k_cache.device))
    _raise_on(rc, "pa_read_kv")
    return out0, out1


def rope_tables(head_dim: int, max_seq_len: int, base: float = 10000.0, device="cuda"):
    """cos / sin tables [max_seq_len, head_dim // 2] in bfloat16 on `device`, computed as
    examples/models/qwen3/kernels/rope.py:4-20 does (float64 frequencies, float32 angles and
    cos / sin, cast to bf16 at the call site attention.py:84-86)."""
    freqs = 1.0 / (base ** (np.arange(0, head_dim, 2)[: (head_dim // 2)] / head_dim))
    ang = np.outer(np.arange(max_seq_len, dtype=np.float32), freqs)
    cos, sin = np.cos(ang, dtype=np.float32), np.sin(ang, dtype=np.float32)
    return (torch.from_numpy(cos).to(device).to(torch.bfloat16), torch.from_numpy(sin).to(device).to(torch.bfloat16))


def qk_norm_rope_kv_write(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, rope_cos, rope_sin, *,
                          q_norm_weight=None, k_norm_weight=None, eps=1e-6, k_scale=None, v_scale=None, out=None):
    """The reference's pre-attention step fused with the paged KV write.

    QK RMSNorm (examples/models/qwen3/kernels/rmsnorm.py:4-21; skipped for a tensor whose weight
    is None), RoPE at absolute positions seq_lens[b] - query_lens[b] + t (rope.py:23-48;
    qwen3/kernels/attention.py:78-97), then `kv_write` of the rotated K and of V.  xq [B, T, Hq, D],
    xk / xv [B, T, Hkv, D] bfloat16; rope_cos / rope_sin [max_pos, D/2] bfloat16 (`rope_tables`).
    Returns the transformed q (`out`, which may be xq itself; padding rows are zero); the pool
    (and its scales for float8) is updated in place.

    xq None: only K and V are done and None is returned; the Q half then rides on the attention
    call as its `q_transform` (a `QTransform` with the same tables), which saves a pass over Q.
    """
    lib = _lib.load()
    for n, t in (("xk", xk), ("xv", xv), ("k_cache", k_cache), ("v_cache", v_cache),
                 ("block_tables", block_tables), ("seq_lens", seq_lens), ("query_lens", query_lens),
                 ("rope_cos", rope_cos), ("rope_sin", rope_sin)):
        _need_device(n, t)
    _check(xk.dim() == 4 and xk.dtype == torch.bfloat16, "xk must be bfloat16 [B, T, Hkv, D]")
    B, T, Hkv, D = xk.shape
    _check(xv.shape == xk.shape and xv.dtype == torch.bfloat16, "xv must match xk")
    if xq is None:
        _check(out is None and q_norm_weight is None, "without xq there is neither out nor q_norm_weight")
        Hq = Hkv
    else:
        _need_device("xq", xq)
        _check(xq.dim() == 4 and xq.dtype == torch.bfloat16 and xq.shape[:2] == (B, T) and xq.shape[3] == D,
               "xq must be bfloat16 [B, T, Hq, D] with xk's B, T and D")
        Hq = xq.shape[2]
    _check(Hq % Hkv == 0, f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    _check(D in (64, 128, 256), f"head_dim {D} must be 64, 128 or 256")
    _check(k_cache.dim() == 4 and tuple(k_cache.shape[2:]) == (Hkv, D), "k_cache must be [num_blocks, block_size, Hkv, D]")
    _check(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype, "v_cache must match k_cache")
    _check(k_cache.dtype in (torch.bfloat16, torch.float8_e4m3fn, torch.int8), f"unsupported pool dtype {k_cache.dtype}")
    num_blocks, block_size = k_cache.shape[:2]
    kv_dtype = _DTYPE_CODE[k_cache.dtype]
    for n, t in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
        _check(t.dim() == 2 and t.shape[1] == D // 2 and t.dtype == torch.bfloat16, f"{n} must be bfloat16 [max_pos, D/2]")
    _check(rope_sin.shape == rope_cos.shape, "rope_sin must match rope_cos")
    for n, t in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if t is not None:
            _need_device(n, t)
            _check(tuple(t.shape) == (D,) and t.dtype == torch.bfloat16, f"{n} must be bfloat16 [D]")
    _check(block_tables.dim() == 2 and block_tables.shape[0] == B and block_tables.dtype == torch.int32,
           "block_tables must be int32 [B, max_blocks]")
    _check(seq_lens.shape == (B,) and seq_lens.dtype == torch.int32, "seq_lens must be int32 [B]")
    _check(query_lens.shape == (B,) and query_lens.dtype == torch.int32, "query_lens must be int32 [B]")
    if kv_dtype in (FP8, I8):
        _check_scales(kv_dtype, k_scale, v_scale, num_blocks, block_size, Hkv, "pool")
    else:
        _check(k_scale is None and v_scale is None, "k_scale / v_scale are for float8 and int8 pools only")
    if xq is not None:
        if out is None:
            out = torch.empty_like(xq)
        else:
            _need_device("out", out)
            _check(out.shape == xq.shape and out.dtype == xq.dtype, "out must match xq")
    _same_device(xk, xq=xq, xv=xv, k_cache=k_cache, v_cache=v_cache, block_tables=block_tables, seq_lens=seq_lens,
                 query_lens=query_lens, rope_cos=rope_cos, rope_sin=rope_sin, q_norm_weight=q_norm_weight,
                 k_norm_weight=k_norm_weight, k_scale=k_scale, v_scale=v_scale, out=out)
    with _on(xk.device):
        rc = lib.pa_qk_norm_rope_kv_write(
            _ptr(xq), _ptr(xk), _ptr(xv), _ptr(out), _ptr(q_norm_weight), _ptr(k_norm_weight), ctypes.c_float(eps),
            _ptr(rope_cos), _ptr(rope_sin), rope_cos.shape[0], _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
            _ptr(block_tables), _ptr(seq_lens), _ptr(query_lens), B, T, Hq, Hkv, D, block_size, block_tables.shape[1],
            num_blocks, kv_dtype, _stream_ptr(xk.device))
    _raise_on(rc, "pa_qk_norm_rope_kv_write")
    return out


def o_proj(x, o_weight, bias=None, *, out=None, workspace=None):
    """Output projection behind the attention call: `np.matmul(output, o_weight)` (+ `o_bias`) of
    examples/models/qwen3/kernels/attention.py:143-147 and examples/models/gpt_oss/kernels/attention.py:155-163.

    x: the attention output, bfloat16, [..., Hq, D] (as `decode` / `prefill` return it) or already
    [..., K] (with a single q head the two readings coincide: `out`'s rank decides, and without `out` x is
    read as [..., K]); o_weight [K, N] bfloat16 with K = Hq * D (the reference's transposed o_proj.weight; a
    tensor-parallel rank passes its own K rows and all-reduces the result itself); bias [N]
    bfloat16 or None.  Returns [..., N] bfloat16 (`out`, if given, is written in place).  Products
    and sums are float32; the result is rounded to bfloat16 once.  Calls of up to 128 rows (decode,
    verify steps) spread K over several workgroups per column slab and need scratch memory for the
    partial sums: a uint8 tensor `workspace` of at least `o_proj_workspace_bytes(M, K, N)` bytes, or,
    by default, a buffer cached per (device, stream).
    """
    lib = _lib.load()
    for n, t in (("x", x), ("o_weight", o_weight)):
        _need_device(n, t)
    _check(x.dtype == torch.bfloat16 and o_weight.dtype == torch.bfloat16, "o_proj supports bfloat16 only")
    _check(o_weight.dim() == 2, "o_weight must be [K, N]")
    K, N = o_weight.shape
    heads_form = x.dim() >= 2 and x.shape[-1] * x.shape[-2] == K      # [..., Hq, D] -> [..., Hq * D]
    flat_form = x.dim() >= 1 and x.shape[-1] == K
    if heads_form and flat_form:
        # one q head (Hq = 1, D = K): both readings fit x.  `out`, when given, says which one the caller means (an engine
        # layer with one q head passes x [B, T, 1, D] and out [B, T, N]); without it x is read as [..., K]
        heads_form = isinstance(out, torch.Tensor) and out.dim() == x.dim() - 1
        flat_form = not heads_form
    if heads_form:
        lead = tuple(x.shape[:-2])
    else:
        _check(flat_form, f"x's last dimension(s) {tuple(x.shape[-2:])} do not give K={K}")
        lead = tuple(x.shape[:-1])
    M = 1
    for d in lead:
        M *= d
    _check(K % 64 == 0, f"K={K} must be a multiple of 64")
    _check(N % 8 == 0, f"N={N} must be a multiple of 8")
    if bias is not None:
        _need_device("bias", bias)
        _check(bias.dtype == torch.bfloat16 and tuple(bias.shape) == (N,), "bias must be bfloat16 [N]")
    _same_device(x, o_weight=o_weight, bias=bias, out=out)
    if out is None:
        out = torch.empty(lead + (N,), dtype=torch.bfloat16, device=x.device)
    else:
        _need_device("out", out)
        _check(tuple(out.shape) == lead + (N,) and out.dtype == torch.bfloat16, f"out must be bfloat16 {lead + (N,)}")
    with _on(x.device):
        stream = _stream_ptr(x.device)
        need = _o_proj_need.get((M, K, N))
        if need is None:
            need = _o_proj_need[(M, K, N)] = int(lib.pa_o_proj_workspace_bytes(M, K, N))
        if workspace is not None:
            _need_device("workspace", workspace)
            _check(workspace.dtype == torch.uint8 and workspace.is_contiguous(), "workspace must be a contiguous uint8 tensor")
            _check(workspace.data_ptr() % 16 == 0, "workspace must be 16-byte aligned")
            _same_device(x, workspace=workspace)
        elif need:
            # (the split form is one more launch: where a step of a few rows is launched call by call and bound by the
            # host it costs 5 us per layer, replayed from a HIP graph it saves 6; it is taken either way, so that the
            # result does not depend on how the call was issued)
            workspace = _workspace(x.device, need, stream)
        rc = lib.pa_o_proj_ws(_ptr(x), _ptr(o_weight), _ptr(bias), _ptr(out), _ptr(workspace),
                              workspace.numel() if workspace is not None else 0, M, K, N, BF16, stream)
    _raise_on(rc, "pa_o_proj")
    return out


class PreparedStep:
    """A `decode_step` / `verify_step` call with its arguments checked and marshalled once, for callers that issue
    the same step on the same tensors again and again (a layer of a decode loop run without a HIP graph: the call
    is then bound by the host, and most of the host's time went into re-checking what had not changed).  `launch()`
    issues it on the current stream and returns `out`.  The step is tied to the storage of every tensor it was
    prepared with (they are kept alive): new values are copied into them, not passed."""
    __slots__ = ("fn", "who", "head", "tail", "need", "workspace", "device", "out", "keep")

    def launch(self):
        stream = _stream_ptr(self.device)
        ws = self.workspace if self.workspace is not None else _workspace(self.device, self.need, stream)
        with _on(self.device):
            rc = self.fn(*self.head, ws.data_ptr(), ws.numel(), *self.tail, stream)
        _raise_on(rc, self.who)
        return self.out

    __call__ = launch


def decode_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, **kw):
    """One decode step of an attention layer in one call; arguments and result as `prepare_decode_step`, which this is
    followed by `launch()`."""
    return prepare_decode_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, **kw).launch()


def prepare_decode_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, *, k_scale=None, v_scale=None,
                        partition_size=512, max_seq_len=None, q_transform=None, k_norm_weight=None, o_weight=None, o_bias=None,
                        out=None, attn_out=None, workspace=None, sinks=None, sliding_window=None) -> PreparedStep:
    """One decode step of an attention layer in one call: the cache update, the attention and, with `o_weight`, the
    output projection -- the decode branch of the reference's attention_kernel as a whole
    (examples/models/qwen3/kernels/attention.py:78-147; examples/models/gpt_oss/kernels/attention.py:85-163).

    Bit for bit the result of `qk_norm_rope_kv_write(None, xk, xv, ...)` (`kv_write` without `q_transform`), then
    `decode(xq, ..., q_transform=...)`, then `o_proj(...)`; a small step over a bfloat16 pool runs as three launches
    instead of five (the new row rides on the decode launch, the split-K merge on the projection's load).

    xq [B, Hq, D], xk / xv [B, Hkv, D]: the step's new token per sequence, before norm and rotation when `q_transform`
    (a `QTransform`: Q's norm weight and the RoPE tables) is given; `k_norm_weight` [D] is K's norm weight (None: K is
    rotated only).  seq_lens counts the new token; query_lens [B] int32 is 1 for the sequences that take one and 0 for
    those that do not.  The pools (and the scales of a float8 pool) are updated in place.
    The step's result (`PreparedStep.out`, what `launch()` returns) is the projected rows [B, N] when `o_weight`
    [Hq * D, N] is given (written to `out` if passed; `attn_out` [B, Hq, D], if passed, also receives the attention
    output), else the attention output [B, Hq, D] (`out`).  Nothing is launched here.
    """
    lib = _lib.load()
    for n, t in (("xq", xq), ("xk", xk), ("xv", xv), ("k_cache", k_cache), ("v_cache", v_cache),
                 ("block_tables", block_tables), ("seq_lens", seq_lens), ("query_lens", query_lens)):
        _need_device(n, t)
    _check(xq.dim() == 3, "xq must be [B, Hq, D]")
    B, Hq, D = xq.shape
    _check(xq.dtype in (torch.float32, torch.bfloat16), f"unsupported xq dtype {xq.dtype}")
    _check_paging(k_cache, v_cache, block_tables, seq_lens, B)
    num_blocks, block_size, Hkv, Dk = k_cache.shape
    _check(Dk == D, f"head_dim mismatch: xq has {D}, cache has {Dk}")
    _check(Hq % Hkv == 0, f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    _check(D in (32, 64, 128, 256), f"head_dim {D} not in (32, 64, 128, 256)")
    _check(tuple(xk.shape) == (B, Hkv, D) and xv.shape == xk.shape and xk.dtype == xq.dtype and xv.dtype == xq.dtype,
           f"xk and xv must be {xq.dtype} [B, Hkv, D] = {(B, Hkv, D)}")
    _check(query_lens.shape == (B,) and query_lens.dtype == torch.int32, "query_lens must be int32 [B]")
    scaled = k_scale is not None or v_scale is not None
    kv_code = _kv_code(k_cache, scaled)
    q_code = _DTYPE_CODE[xq.dtype]
    if kv_code in (FP8, I8):
        _check(q_code == BF16, f"{'fp8' if kv_code == FP8 else 'int8'} KV needs bfloat16 rows")
        _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv)
        _check(kv_code == FP8 or verify_supported(1, D, block_size),
               f"int8 KV needs head_dim 64 or 128 and a power-of-two block size >= 16 (D={D}, block_size={block_size})")
    else:
        _check(kv_code == q_code, f"KV dtype {k_cache.dtype} does not match the rows' dtype {xq.dtype}")
        _check(not scaled, "k_scale/v_scale are only valid with an fp8 or int8 KV cache")
    sinks, win = _check_variant(sinks, sliding_window, Hq, xq)
    _check(isinstance(partition_size, int) and partition_size > 0, "partition_size must be a positive int")
    cap = block_tables.shape[1] * block_size
    msl = cap if max_seq_len is None else int(max_seq_len)
    _check(0 < msl <= cap, f"max_seq_len {msl} outside (0, {cap}]")
    if k_norm_weight is not None:
        _need_device("k_norm_weight", k_norm_weight)
        _check(q_transform is not None, "k_norm_weight comes with q_transform")
        _check(tuple(k_norm_weight.shape) == (D,) and k_norm_weight.dtype == torch.bfloat16, "k_norm_weight must be bfloat16 [D]")
    N = 0
    if o_weight is not None:
        _need_device("o_weight", o_weight)
        _check(xq.dtype == torch.bfloat16 and o_weight.dtype == torch.bfloat16, "the output projection supports bfloat16 only")
        _check(o_weight.dim() == 2 and o_weight.shape[0] == Hq * D, f"o_weight must be [Hq * D = {Hq * D}, N]")
        N = o_weight.shape[1]
        _check((Hq * D) % 64 == 0 and N % 8 == 0, f"Hq * D = {Hq * D} must be a multiple of 64 and N = {N} of 8")
        if o_bias is not None:
            _need_device("o_bias", o_bias)
            _check(o_bias.dtype == torch.bfloat16 and tuple(o_bias.shape) == (N,), "o_bias must be bfloat16 [N]")
        if out is None:
            out = torch.empty((B, N), dtype=torch.bfloat16, device=xq.device)
        else:
            _need_device("out", out)
            _check(tuple(out.shape) == (B, N) and out.dtype == torch.bfloat16, f"out must be bfloat16 {(B, N)}")
        if attn_out is not None:
            _need_device("attn_out", attn_out)
            _check(attn_out.shape == xq.shape and attn_out.dtype == xq.dtype, "attn_out must match xq in shape and dtype")
    else:
        _check(o_bias is None and attn_out is None, "o_bias and attn_out come with o_weight (without it `out` is the attention output)")
        if out is None:
            out = torch.empty_like(xq)
        else:
            _need_device("out", out)
            _check(out.shape == xq.shape and out.dtype == xq.dtype, "out must match xq in shape and dtype")
        attn_out = out
    _same_device(xq, xk=xk, xv=xv, k_cache=k_cache, v_cache=v_cache, block_tables=block_tables, seq_lens=seq_lens,
                 query_lens=query_lens, k_scale=k_scale, v_scale=v_scale, out=out, attn_out=attn_out, o_weight=o_weight,
                 o_bias=o_bias, k_norm_weight=k_norm_weight)
    key = (B, Hq, Hkv, D, block_size, msl, partition_size, N, q_code, kv_code)
    need = _decode_step_need.get(key)
    if need is None:
        with _on(xq.device):
            need = _decode_step_need[key] = int(lib.pa_decode_step_workspace_bytes(*key))
    if workspace is not None:
        _need_device("workspace", workspace)
        _check(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0,
               "workspace must be a contiguous, 16-byte aligned uint8 tensor")
        _check(workspace.numel() >= need, f"workspace needs {need} bytes")
    qt_keep, qt_ptr = _qt_arg(q_transform, D, xq)
    addr = lambda t: None if t is None else t.data_ptr()
    nkv = _lib.NewKvStruct(addr(xk), addr(xv), addr(k_norm_weight), addr(query_lens))
    proj = None if o_weight is None else _lib.OutProjStruct(addr(o_weight), addr(o_bias), addr(out), N)
    st = PreparedStep()
    st.fn, st.who, st.need, st.workspace, st.device, st.out = lib.pa_decode_step, "pa_decode_step", need, workspace, xq.device, out
    st.head = (_ptr(xq), ctypes.addressof(nkv), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
               _ptr(block_tables), _ptr(seq_lens), _ptr(attn_out), None if proj is None else ctypes.addressof(proj))
    st.tail = (B, Hq, Hkv, D, block_size, block_tables.shape[1], num_blocks, msl,
               float(scale), partition_size, q_code, kv_code, _ptr(sinks), win, qt_ptr)
    # everything an address above points into stays alive with the step
    st.keep = (nkv, proj, qt_keep, xq, xk, xv, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, query_lens,
               attn_out, out, sinks, k_norm_weight, o_weight, o_bias, q_transform)
    return st


_decode_step_need = {}


def verify_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, **kw):
    """A speculative verify step of an attention layer in one call; arguments and result as `prepare_verify_step`,
    which this is followed by `launch()`."""
    return prepare_verify_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, **kw).launch()


def prepare_verify_step(xq, xk, xv, k_cache, v_cache, block_tables, seq_lens, query_lens, scale, *, k_scale=None, v_scale=None,
                        max_seq_len=None, q_transform=None, k_norm_weight=None, o_weight=None, o_bias=None, out=None,
                        attn_out=None, workspace=None, sinks=None, sliding_window=None) -> PreparedStep:
    """A speculative verify step of an attention layer in one call: `decode_step` for up to 64 new tokens per sequence
    (examples/models/gpt_oss/kernels/attention.py:80-163 with seq_len = K + 1; peagle/speculate.py:137-202).

    Bit for bit `qk_norm_rope_kv_write(None, xk, xv, ...)` (`kv_write` without `q_transform`), `verify(xq, ...)`,
    `o_proj(...)`.  xq [B, T, Hq, D], xk / xv [B, T, Hkv, D] bfloat16; query_lens [B]: new tokens per sequence (rows
    t >= query_lens[b] are padding: zero attention output, bias after the projection).  The step's result is
    [B, T, N] with `o_weight`, else the attention output [B, T, Hq, D].  Nothing is launched here."""
    lib = _lib.load()
    for n, t in (("xq", xq), ("xk", xk), ("xv", xv), ("k_cache", k_cache), ("v_cache", v_cache),
                 ("block_tables", block_tables), ("seq_lens", seq_lens), ("query_lens", query_lens)):
        _need_device(n, t)
    _check(xq.dim() == 4, "xq must be [B, T, Hq, D]")
    B, T, Hq, D = xq.shape
    _check(xq.dtype == torch.bfloat16, "verify_step supports bfloat16 rows only")
    _check_paging(k_cache, v_cache, block_tables, seq_lens, B)
    num_blocks, block_size, Hkv, Dk = k_cache.shape
    _check(Dk == D, f"head_dim mismatch: xq has {D}, cache has {Dk}")
    _check(Hq % Hkv == 0, f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    _check(verify_supported(T, D, block_size),
           f"the verify kernel needs T <= 64, head_dim 64 or 128 and a power-of-two block size >= 16 (T={T}, D={D}, block_size={block_size})")
    _check(tuple(xk.shape) == (B, T, Hkv, D) and xv.shape == xk.shape and xk.dtype == xq.dtype and xv.dtype == xq.dtype,
           f"xk and xv must be bfloat16 [B, T, Hkv, D] = {(B, T, Hkv, D)}")
    _check(query_lens.shape == (B,) and query_lens.dtype == torch.int32, "query_lens must be int32 [B]")
    scaled = k_scale is not None or v_scale is not None
    kv_code = _kv_code(k_cache, scaled)
    _check(kv_code in (BF16, FP8, I8), "verify_step needs a bfloat16, fp8 or int8 KV cache")
    if kv_code in (FP8, I8):
        _check_scales(kv_code, k_scale, v_scale, num_blocks, block_size, Hkv)
    else:
        _check(not scaled, "k_scale/v_scale are only valid with an fp8 or int8 KV cache")
    sinks, win = _check_variant(sinks, sliding_window, Hq, xq)
    cap = block_tables.shape[1] * block_size
    msl = 0 if max_seq_len is None else int(max_seq_len)
    _check(max_seq_len is None or 0 < msl <= cap, f"max_seq_len {msl} outside (0, {cap}]")
    if k_norm_weight is not None:
        _need_device("k_norm_weight", k_norm_weight)
        _check(q_transform is not None, "k_norm_weight comes with q_transform")
        _check(tuple(k_norm_weight.shape) == (D,) and k_norm_weight.dtype == torch.bfloat16, "k_norm_weight must be bfloat16 [D]")
    N = 0
    if o_weight is not None:
        _need_device("o_weight", o_weight)
        _check(o_weight.dtype == torch.bfloat16 and o_weight.dim() == 2 and o_weight.shape[0] == Hq * D,
               f"o_weight must be bfloat16 [Hq * D = {Hq * D}, N]")
        N = o_weight.shape[1]
        _check((Hq * D) % 64 == 0 and N % 8 == 0, f"Hq * D = {Hq * D} must be a multiple of 64 and N = {N} of 8")
        if o_bias is not None:
            _need_device("o_bias", o_bias)
            _check(o_bias.dtype == torch.bfloat16 and tuple(o_bias.shape) == (N,), "o_bias must be bfloat16 [N]")
        if out is None:
            out = torch.empty((B, T, N), dtype=torch.bfloat16, device=xq.device)
        else:
            _need_device("out", out)
            _check(tuple(out.shape) == (B, T, N) and out.dtype == torch.bfloat16, f"out must be bfloat16 {(B, T, N)}")
        if attn_out is not None:
            _need_device("attn_out", attn_out)
            _check(attn_out.shape == xq.shape and attn_out.dtype == xq.dtype, "attn_out must match xq in shape and dtype")
    else:
        _check(o_bias is None and attn_out is None, "o_bias and attn_out come with o_weight (without it `out` is the attention output)")
        if out is None:
            out = torch.empty_like(xq)
        else:
            _need_device("out", out)
            _check(out.shape == xq.shape and out.dtype == xq.dtype, "out must match xq in shape and dtype")
        attn_out = out
    _same_device(xq, xk=xk, xv=xv, k_cache=k_cache, v_cache=v_cache, block_tables=block_tables, seq_lens=seq_lens,
                 query_lens=query_lens, k_scale=k_scale, v_scale=v_scale, out=out, attn_out=attn_out, o_weight=o_weight,
                 o_bias=o_bias, k_norm_weight=k_norm_weight)
    key = ("v", B, T, Hq, D, N)
    need = _decode_step_need.get(key)
    if need is None:
        with _on(xq.device):
            need = _decode_step_need[key] = int(lib.pa_verify_step_workspace_bytes(B, T, Hq, D, N))
    if workspace is not None:
        _need_device("workspace", workspace)
        _check(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0,
               "workspace must be a contiguous, 16-byte aligned uint8 tensor")
        _check(workspace.numel() >= need, f"workspace needs {need} bytes")
    qt_keep, qt_ptr = _qt_arg(q_transform, D, xq)
    addr = lambda t: None if t is None else t.data_ptr()
    nkv = _lib.NewKvStruct(addr(xk), addr(xv), addr(k_norm_weight), addr(query_lens))
    proj = None if o_weight is None else _lib.OutProjStruct(addr(o_weight), addr(o_bias), addr(out), N)
    st = PreparedStep()
    st.fn, st.who, st.need, st.workspace, st.device, st.out = lib.pa_verify_step, "pa_verify_step", need, workspace, xq.device, out
    st.head = (_ptr(xq), ctypes.addressof(nkv), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
               _ptr(block_tables), _ptr(seq_lens), _ptr(attn_out), None if proj is None else ctypes.addressof(proj))
    st.tail = (B, T, Hq, Hkv, D, block_size, block_tables.shape[1], num_blocks, msl,
               float(scale), kv_code, _ptr(sinks), win, qt_ptr)
    st.keep = (nkv, proj, qt_keep, xq, xk, xv, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, query_lens,
               attn_out, out, sinks, k_norm_weight, o_weight, o_bias, q_transform)
    return st
def o_proj_workspace_bytes(M: int, K: int, N: int) -> int:
    """Scratch bytes `o_proj` would use for a call of M rows (0 for shapes that take none)."""
    return int(_lib.load().pa_o_proj_workspace_bytes(int(M), int(K), int(N)))


def default_scale(head_dim: int) -> float:
    """1 / sqrt(head_dim) in float32, as examples/models/qwen3/kernels/attention.py:119."""
    return float(np.float32(1.0) / np.float32(math.sqrt(head_dim)))
