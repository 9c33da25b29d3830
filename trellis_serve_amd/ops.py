"""Torch-facing wrappers of the C-ABI: device tensors in, device tensors out, every launch on the current stream.

These mirror the building blocks of the reference's Marlin backend (cuda/src/sglang_exl3/kernels/marlin.py:138-190)
and ExLlamaV3's reconstruct (cuda/src/sglang_exl3/kernels/reference.py:71-76), with the same argument meaning.
Nothing here computes on the CPU: a missing library raises ExtensionMissing.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

CODEBOOK_ID = {"3inst": 0, "mcg": 1, "mul1": 2}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    """The current stream's handle, without the Stream object around it (0.15 us instead of 2.0 per call)."""
    if device.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {device}")
    return torch._C._cuda_getCurrentRawStream(_dev_index(device))


def bits_of(trellis: torch.Tensor) -> int:
    """K from the trellis last dim (16 K int16 per tile; core/src/trellis_core/format/spec.py:58-61)."""
    words = trellis.shape[-1]
    if words % 16:
        raise ValueError(f"trellis last dim {words} is not 16*K")
    return words // 16


def _check_trellis(t: torch.Tensor) -> tuple[int, int, int]:
    shape = t.shape
    if t.dtype != torch.int16 or len(shape) != 3 or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"trellis must be a contiguous CUDA int16 [k/16, n/16, 16K] tensor, got {t.dtype} "
                         f"{tuple(shape)} on {t.device}")
    rows, cols, words = shape
    return rows * 16, cols * 16, words // 16 if words % 16 == 0 else bits_of(t)


def _half(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA fp16 tensor, got {t.dtype} on {t.device}")
    return t


class WorkspaceTooSmall(RuntimeError):
    """A call inside HIP-graph capture needs more workspace than was reserved (nothing may allocate there)."""


class _Workspace:
    """The per-device scratch of one kind of launch (split counters, rotated activations, fp32 partials).

    A workspace only ever grows by replacement while no captured graph can hold its address.  Once it has been used
    inside a graph capture it is never freed or replaced: a later eager call that needs more runs on a temporary
    buffer of its own (as the reference's run does past its reserved rows, cuda/src/sglang_exl3/kernels/marlin.py:
    86-89), and a capture that needs more raises WorkspaceTooSmall.  After `reserve_*` the workspace keeps its
    reserved size the same way, so an engine that reserves for its largest batch at load time never allocates on the
    serving path (cuda/src/sglang_exl3/kernels/base.py:74-76)."""

    def __init__(self, kind: str, zeroed: bool):
        self.kind, self.zeroed = kind, zeroed
        self.buf: torch.Tensor | None = None
        self.reserved = False   # sized by reserve_*: later calls beyond it use a temporary buffer
        self.captured = False   # used inside a graph capture: the address must never change

    def _alloc(self, nbytes: int, device: torch.device) -> torch.Tensor:
        # counters must start at zero (every call leaves them there); the KV workspace holds only fully written data
        make = torch.zeros if self.zeroed else torch.empty
        return make(max(int(nbytes), 256), dtype=torch.uint8, device=device)

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor:
        capturing = torch.cuda.is_current_stream_capturing()
        if self.buf is not None and self.buf.numel() >= nbytes:
            self.captured |= capturing
            return self.buf
        have = 0 if self.buf is None else self.buf.numel()
        if capturing:
            raise WorkspaceTooSmall(f"{self.kind} workspace on {device} holds {have} bytes, a call inside graph capture "
                                    f"needs {nbytes}: call ops.reserve_{self.kind}(...) for the largest shape before "
                                    f"capturing")
        if self.captured or self.reserved:
            return self._alloc(nbytes, device)   # one-off: the reserved buffer keeps its address
        self.buf = self._alloc(nbytes, device)
        return self.buf

    def reserve(self, device: torch.device, nbytes: int) -> None:
        if self.buf is None or self.buf.numel() < nbytes:
            if self.captured:
                raise WorkspaceTooSmall(f"{self.kind} workspace on {device} is held by a captured graph; reserve "
                                        f"{nbytes} bytes before the first capture")
            self.buf = self._alloc(nbytes, device)
        self.reserved = True


_KINDS = {"linear": True, "prefill": True, "moe": True, "moe_stage": True, "kv": False}
_workspaces: dict[tuple[str, int], _Workspace] = {}


def _dev_index(device: torch.device) -> int:
    index = device.index
    return index if index is not None else torch.cuda.current_device()


def _elsewhere(device: torch.device) -> bool:
    """Whether another device is current: plans that follow the current device's CU count (the decode-GEMM's, past 32
    rows of a linear) are then sized and launched with `device` current."""
    return _dev_index(device) != torch.cuda.current_device()


_initialised: set[int] = set()


def _ws(kind: str, device: torch.device) -> _Workspace:
    idx = _dev_index(device)
    if idx not in _initialised and not torch.cuda.is_current_stream_capturing():
        # the device check, and the probe of the workgroup -> XCD assignment that lets split-K chains stay in one
        # XCD's L2 (the reference's init_device, cuda/csrc/exl3_marlin.cu:537); a workspace is first taken (or
        # reserved) before any capture
        init_device(idx)
        _initialised.add(idx)
    key = (kind, idx)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = _Workspace(kind, _KINDS[kind])
    return ws


def workspace(device: torch.device, nbytes: int, kind: str = "linear") -> torch.Tensor:
    """The per-device workspace of `kind` ("linear", "prefill", "moe", "kv") holding at least `nbytes`."""
    if device.index is None or device.type != "cuda":
        device = torch.device("cuda", _dev_index(device))
    return _ws(kind, device).get(device, nbytes)


def release_workspaces() -> None:
    """Drops every workspace (tests; an engine that has captured graphs must keep them)."""
    _workspaces.clear()


def _max_need(fn, max_rows: int) -> int:
    """The largest workspace any row count 1..max_rows needs (split plans do not grow monotonically with rows)."""
    return max(fn(r) for r in range(1, max(1, int(max_rows)) + 1))


def reserve_linear(device: torch.device, max_rows: int, k: int, n_total: int, K: int) -> None:
    """Reserves the decode-GEMV workspace for every call of up to `max_rows` rows on a group of input width k and
    n_total output columns at bitrate K (the reference reserves its scratch at load, kernels/marlin.py:24-33)."""
    lib = _lib.load()
    dev = torch.device("cuda", _dev_index(device))
    with torch.cuda.device(dev):   # the plan depends on the device's CU count
        need = _max_need(lambda r: lib.exl3_linear_workspace_bytes(r, k, n_total, K), max_rows)
    _ws("linear", dev).reserve(dev, need)


def reserve_prefill(device: torch.device, max_rows: int, k: int, n_total: int, nshards: int) -> None:
    """Reserves the decode-GEMM workspace for every call of up to `max_rows` rows."""
    lib = _lib.load()
    dev = torch.device("cuda", _dev_index(device))
    with torch.cuda.device(dev):   # the plan depends on the device's CU count
        need = lib.exl3_prefill_workspace_bytes(max(1, int(max_rows)), k, n_total, nshards)
    _ws("prefill", dev).reserve(dev, need)


def reserve_moe(device: torch.device, max_tokens: int, top_k: int, num_experts: int, hidden: int, inter: int,
                K_gate_up: int, K_down: int) -> None:
    """Reserves the MoE workspace for every call of up to `max_tokens` tokens."""
    lib = _lib.load()
    dev = torch.device("cuda", _dev_index(device))
    _ws("moe", dev).reserve(dev, lib.exl3_moe_workspace_bytes(max(1, int(max_tokens)), top_k, num_experts, hidden, inter,
                                                              K_gate_up, K_down))


def moe_align_capacity(slots: int, num_experts: int, block: int) -> tuple[int, int]:
    """(sorted_ids entries, expert_ids blocks) that moe_align allocates for `slots` routed slots."""
    cap = slots + num_experts * (block - 1)
    return cap, -(-cap // block)


def reserve_moe_stage(device: torch.device, max_slots: int, k: int, n: int, shards: int, num_experts: int,
                      block: int) -> None:
    """Reserves the grouped-GEMM workspace of the per-launch MoE stages (moe_gemm) for every call of up to `max_slots`
    rows routed by moe_align with `num_experts` experts and this block size, so a captured stage chain never
    allocates."""
    lib = _lib.load()
    dev = torch.device("cuda", _dev_index(device))
    need = _max_need(lambda r: lib.exl3_moe_gemm_workspace_bytes(r, k, n, shards,
                                                                 moe_align_capacity(r, num_experts, block)[1]),
                     max_slots)
    _ws("moe_stage", dev).reserve(dev, need)


def reserve_kv(device: torch.device, max_batch: int, num_q_heads: int, num_kv_heads: int, max_pages: int) -> None:
    """Reserves the KV decode-attention workspace for batches of up to `max_batch` sequences of up to `max_pages`
    pages (a smaller batch can take more page chunks per sequence, so every batch size is sized; fewer pages never
    need more)."""
    lib = _lib.load()
    dev = torch.device("cuda", _dev_index(device))
    _ws("kv", dev).reserve(dev, _max_need(
        lambda b: lib.exl3_kv_decode_workspace_bytes(b, num_q_heads, num_kv_heads, max_pages), max_batch))


def reserve_workspace(device: torch.device, rows: int, k: int, n_total: int, K: int) -> None:
    """Older name of reserve_linear."""
    reserve_linear(device, rows, k, n_total, K)


def _check_out(out: torch.Tensor, shape: tuple, like: torch.Tensor, dtypes=(torch.float16, torch.bfloat16)) -> None:
    """A caller-supplied output must be exactly what the kernels write: the C-ABI only sees a pointer."""
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(shape)}")
    if out.dtype not in dtypes:
        raise ValueError(f"out must be one of {[str(d) for d in dtypes]}, got {out.dtype}")
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    if out.device != like.device:
        raise ValueError(f"out is on {out.device}, the inputs on {like.device}")


def init_device(index: int) -> None:
    _lib.check(_lib.load().exl3_init_device(int(index)), "exl3_init_device")


def reconstruct(trellis: torch.Tensor, codebook: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """W_inner fp16 [k, n], bit-identical to trellis_core.reference.reconstruct_inner (reference.py:102-115)."""
    k, n, K = _check_trellis(trellis)
    if out is None:
        out = torch.empty((k, n), dtype=torch.float16, device=trellis.device)
    if out.shape != (k, n) or out.dtype != torch.float16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous fp16 [k, n] tensor")
    _lib.check(_lib.load().exl3_reconstruct(trellis.data_ptr(), k, n, K, int(codebook), out.data_ptr(),
                                            _stream(trellis.device)), "reconstruct")
    return out


def repack_trellis(trellis: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The trellis in the load-time layout (LAYOUT_BLOCKS; the reference's repack_trellis,
    cuda/csrc/exl3_marlin.cu:344-381): the same bytes per tile, each (128-column block, 128-row block) unit of 64
    tiles one contiguous run.  Same shape and dtype as the stored tensor; `out` must not be the input."""
    return _trellis_relayout(trellis, out, "exl3_repack_trellis")


def unpack_trellis(packed: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Inverse of repack_trellis: the stored layout back, bit for bit (the reference's unpack_trellis,
    exl3_marlin.cu:384-408)."""
    return _trellis_relayout(packed, out, "exl3_unpack_trellis")


def _trellis_relayout(t: torch.Tensor, out: torch.Tensor | None, entry: str) -> torch.Tensor:
    k, n, K = _check_trellis(t)
    if out is None:
        out = torch.empty_like(t)
    if out.shape != t.shape or out.dtype != torch.int16 or not out.is_contiguous() or out.device != t.device:
        raise ValueError(f"out must be a contiguous int16 {tuple(t.shape)} tensor on {t.device}")
    if out.data_ptr() == t.data_ptr():
        raise ValueError(f"{entry}: out must not be the input")
    _lib.check(getattr(_lib.load(), entry)(t.data_ptr(), k, n, K, out.data_ptr(), _stream(t.device)), entry)
    return out


def had_in_group(x: torch.Tensor, suh_cat: torch.Tensor, xh: torch.Tensor | None = None) -> torch.Tensor:
    """xh[s] = fp16(Had128(fp16(x) * suh_cat[s])) for all shards: x fp16|bf16 [rows, k] -> fp16 [shards*rows, k]
    (kernels/marlin.py:138-146)."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous fp16/bf16 [rows, k] tensor")
    rows, k = x.shape
    suh_cat = _half(suh_cat, "suh_cat")
    shards = suh_cat.numel() // k
    if shards * k != suh_cat.numel():
        raise ValueError(f"suh_cat has {suh_cat.numel()} values, not a multiple of k = {k}")
    if xh is None:
        xh = torch.empty((shards * rows, k), dtype=torch.float16, device=x.device)
    _lib.check(_lib.load().exl3_had_in_group(x.data_ptr(), int(x.dtype == torch.bfloat16), rows, k,
                                             suh_cat.data_ptr(), shards, xh.data_ptr(), _stream(x.device)),
               "had_in_group")
    return xh


def had_out_into(y: torch.Tensor, svh: torch.Tensor, out: torch.Tensor, col0: int) -> None:
    """out[:, col0:col0+n] = fp16(Had128(y)) * svh in out's dtype (kernels/marlin.py:149-151)."""
    y = _half(y, "y")
    rows, n = y.shape
    if out.dtype not in (torch.float16, torch.bfloat16) or out.dim() != 2 or out.stride(1) != 1:
        raise ValueError("out must be an fp16/bf16 [rows, N] tensor with unit column stride")
    if out.shape[0] != rows or col0 + n > out.shape[1]:
        raise ValueError(f"out {tuple(out.shape)} cannot hold columns {col0}..{col0 + n} of {rows} rows")
    _lib.check(_lib.load().exl3_had_out_into(y.data_ptr(), rows, n, _half(svh, "svh").data_ptr(), out.data_ptr(),
                                             int(out.dtype == torch.bfloat16), out.stride(0), int(col0),
                                             _stream(y.device)), "had_out_into")


def gemm_rotated(xh: torch.Tensor, trellis: torch.Tensor, codebook: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """xh @ W_inner in the rotated basis, fp32 accumulation, fp16 out; identity rows read W_inner out exactly
    (kernels/marlin.py:153-159).  Below 65 rows the decode-GEMV serves the rows, from 65 rows the prefill
    decode-GEMM."""
    k, n, K = _check_trellis(trellis)
    xh = _half(xh, "xh")
    if xh.dim() != 2 or xh.shape[1] != k:
        raise ValueError(f"xh must be [rows, {k}]")
    rows = xh.shape[0]
    if rows > 64 and _elsewhere(xh.device):
        with torch.cuda.device(xh.device):
            return gemm_rotated(xh, trellis, codebook, out)
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float16, device=xh.device)
    _check_out(out, (rows, n), xh, (torch.float16,))
    lib = _lib.load()
    ws = workspace(xh.device, lib.exl3_gemm_rotated_workspace_bytes(rows, k, n, K))
    _lib.check(lib.exl3_gemm_rotated(xh.data_ptr(), rows, k, trellis.data_ptr(), n, K, int(codebook),
                                     out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(xh.device)), "gemm_rotated")
    return out


def _shards(trellis: list[torch.Tensor], suh: list[torch.Tensor], svh: list[torch.Tensor], device: torch.device,
            layout: int = _lib.LAYOUT_STORED):
    if not (1 <= len(trellis) <= _lib.MAX_SHARDS) or not (len(trellis) == len(suh) == len(svh)):
        raise ValueError(f"1..{_lib.MAX_SHARDS} shards with one trellis, suh and svh each")
    arr = (_lib.Exl3Shard * len(trellis))()
    k0 = K0 = None
    for i, (t, su, sv) in enumerate(zip(trellis, suh, svh)):
        k, n, K = _check_trellis(t)
        if k0 is None:
            k0, K0 = k, K
        if k != k0 or K != K0:
            raise ValueError("all shards of a group share the input width k and the bitrate K")
        if _half(su, "suh").numel() != k or _half(sv, "svh").numel() != n:
            raise ValueError(f"shard {i}: suh/svh sizes {su.numel()}/{sv.numel()} != {k}/{n}")
        if not (t.device == su.device == sv.device == device):
            raise ValueError(f"shard {i}: tensors on {t.device}/{su.device}/{sv.device}, x on {device}")
        a = arr[i]
        a.trellis, a.suh, a.svh, a.n, a.layout = t.data_ptr(), su.data_ptr(), sv.data_ptr(), n, int(layout)
    return arr, k0, K0


def _rows2d(x: torch.Tensor, k: int) -> torch.Tensor:
    """The rows of x [..., k] as a contiguous 2-D tensor (x itself where it is one)."""
    rows2d = x if x.dim() == 2 and x.is_contiguous() else x.reshape(-1, x.shape[-1]).contiguous()
    if rows2d.shape[1] != k:
        raise ValueError(f"x has {rows2d.shape[1]} features, the group expects {k}")
    return rows2d


def _out2d(x: torch.Tensor, rows: int, n_total: int, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty((rows, n_total), dtype=x.dtype, device=x.device)
    _check_out(out, (rows, n_total), x)
    return out


def _like_x(out: torch.Tensor, x: torch.Tensor, n_total: int) -> torch.Tensor:
    return out if x.dim() == 2 else out.view(*x.shape[:-1], n_total)


def linear(x: torch.Tensor, trellis: list[torch.Tensor], suh: list[torch.Tensor], svh: list[torch.Tensor],
           codebook: int, out: torch.Tensor | None = None, layout: int = _lib.LAYOUT_STORED) -> torch.Tensor:
    """Fused group: y[..., sum n_s] = concat_s(Had(Had(x * suh_s) @ W_s) * svh_s), x fp16|bf16 [..., k], y in x's
    dtype (exl3_linear_marlin_multi_out, cuda/csrc/exl3_marlin.cu:507-527)."""
    bf16 = x.dtype == torch.bfloat16
    if not bf16 and x.dtype != torch.float16:
        raise ValueError(f"x must be fp16 or bf16, got {x.dtype}")
    device = x.device
    arr, k, K = _shards(trellis, suh, svh, device, layout)
    rows2d = _rows2d(x, k)
    rows = rows2d.shape[0]
    if rows > 32 and _elsewhere(device):
        with torch.cuda.device(device):
            return linear(x, trellis, suh, svh, codebook, out, layout)
    n_total = sum([a.n for a in arr])
    out = _out2d(x, rows, n_total, out)
    lib = _lib.load()
    ws = workspace(device, lib.exl3_linear_workspace_bytes(rows, k, n_total, K))
    _lib.check(lib.exl3_linear(rows2d.data_ptr(), int(bf16), rows, k, arr, len(arr), K, int(codebook), out.data_ptr(),
                               int(out.dtype == torch.bfloat16), ws.data_ptr(), ws.numel(), _stream(device)), "linear")
    return _like_x(out, x, n_total)


def linear_prefill(x: torch.Tensor, trellis: list[torch.Tensor], suh: list[torch.Tensor], svh: list[torch.Tensor],
                   codebook: int, out: torch.Tensor | None = None, layout: int = _lib.LAYOUT_STORED) -> torch.Tensor:
    """Many-row form of `linear`: input rotations into a per-device workspace, then the fused decode-GEMM (weights
    decoded into registers, fp16 MFMA).  Same result contract as `linear` (the reference's prefill branch,
    cuda/src/sglang_exl3/runtime/ops.py:87-95)."""
    bf16 = x.dtype == torch.bfloat16
    if not bf16 and x.dtype != torch.float16:
        raise ValueError(f"x must be fp16 or bf16, got {x.dtype}")
    device = x.device
    arr, k, K = _shards(trellis, suh, svh, device, layout)
    rows2d = _rows2d(x, k)
    rows = rows2d.shape[0]
    if _elsewhere(device):
        with torch.cuda.device(device):
            return linear_prefill(x, trellis, suh, svh, codebook, out, layout)
    n_total = sum([a.n for a in arr])
    out = _out2d(x, rows, n_total, out)
    lib = _lib.load()
    ws = workspace(device, lib.exl3_prefill_workspace_bytes(rows, k, n_total, len(arr)), "prefill")
    _lib.check(lib.exl3_linear_prefill(rows2d.data_ptr(), int(bf16), rows, k, arr, len(arr), K, int(codebook),
                                       out.data_ptr(), int(out.dtype == torch.bfloat16), ws.data_ptr(), ws.numel(),
                                       _stream(device)), "linear_prefill")
    return _like_x(out, x, n_total)


MOE_TENSORS = ("gate_trellis", "up_trellis", "down_trellis", "gate_suh", "gate_svh", "up_suh", "up_svh", "down_suh",
               "down_svh")


def _expert_stacks(experts: dict[str, torch.Tensor], H: int, device: torch.device) -> tuple[int, int, int, int]:
    """Checks one set of stacked expert tensors (MOE_TENSORS); returns (E, inter, K gate/up, K down)."""
    gt, ut, dt = experts["gate_trellis"], experts["up_trellis"], experts["down_trellis"]
    if any(t.dim() != 4 or t.dtype != torch.int16 for t in (gt, ut, dt)):
        raise ValueError("stacked trellis tensors must be int16 [E, k/16, n/16, 16K]")
    E, I = gt.shape[0], gt.shape[2] * 16
    if ut.shape != gt.shape:
        raise ValueError(f"gate {tuple(gt.shape)} and up {tuple(ut.shape)} must have one shape and bitrate")
    if gt.shape[1] * 16 != H or tuple(dt.shape[:3]) != (E, I // 16, H // 16):
        raise ValueError(f"expert shapes {tuple(gt.shape)} / {tuple(dt.shape)} do not match H = {H}")
    sizes = {"gate_suh": H, "up_suh": H, "gate_svh": I, "up_svh": I, "down_suh": I, "down_svh": H}
    for name in MOE_TENSORS:
        t = experts[name]
        if not (t.is_cuda and t.is_contiguous()) or t.shape[0] != E or t.device != device:
            raise ValueError(f"{name} must be a contiguous tensor with {E} experts on {device}")
        if name in sizes and (t.dtype != torch.float16 or tuple(t.shape) != (E, sizes[name])):
            raise ValueError(f"{name} must be fp16 [{E}, {sizes[name]}], got {t.dtype} {tuple(t.shape)}")
    return E, I, bits_of(gt), bits_of(dt)


def _routing(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor):
    T = x.shape[0]
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or tuple(topk_weights.shape) != tuple(topk_ids.shape):
        raise ValueError(f"topk_ids {tuple(topk_ids.shape)} and topk_weights {tuple(topk_weights.shape)} must both be "
                         f"[{T}, top_k]")
    if topk_ids.dtype not in (torch.int32, torch.int64) or topk_ids.device != x.device \
            or topk_weights.device != x.device:
        raise ValueError("topk_ids must be int32/int64 and both routing tensors on x's device")
    return topk_ids.to(torch.int32).contiguous(), topk_weights.to(torch.float32).contiguous()


def moe_forward(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, experts: dict[str, torch.Tensor],
                codebook: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Routed SiLU-gated EXL3 MoE layer (cuda/src/sglang_exl3/kernels/marlin_moe.py:272-294).
    x fp16|bf16 [T, H]; topk_ids [T, top_k] (int32 or int64); topk_weights fp32 [T, top_k]; `experts` holds the
    stacked tensors named in MOE_TENSORS (trellis int16 [E, k/16, n/16, 16K], scales fp16 [E, k] / [E, n]).
    Gate and up share one bitrate, down may have another (cuda/src/sglang_exl3/kernels/reference.py:123-149)."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        raise ValueError("x must be a 2-D fp16/bf16 tensor")
    T, H = x.shape
    E, I, K_gu, K_dn = _expert_stacks(experts, H, x.device)
    ids, w = _routing(x, topk_ids, topk_weights)
    top_k = ids.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    _check_out(out, (T, H), x)
    lib = _lib.load()
    ws = workspace(x.device, lib.exl3_moe_workspace_bytes(T, top_k, E, H, I, K_gu, K_dn), "moe")
    wts = _lib.Exl3MoeWeights(*[experts[n].data_ptr() for n in MOE_TENSORS])
    _lib.check(lib.exl3_moe_forward(x.contiguous().data_ptr(), int(x.dtype == torch.bfloat16), T, H, ids.data_ptr(),
                                    w.data_ptr(), top_k, E, I, ctypes.byref(wts), K_gu, K_dn, int(codebook),
                                    out.data_ptr(), int(out.dtype == torch.bfloat16), ws.data_ptr(), ws.numel(),
                                    _stream(x.device)),
               "moe_forward")
    return out


def moe_forward_classes(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                        classes: list[tuple[dict[str, torch.Tensor], torch.Tensor]], num_experts: int, codebook: int,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """moe_forward for a layer whose experts come in up to two K classes (the reference's MixedPack / run_mixed,
    cuda/src/sglang_exl3/kernels/marlin_moe.py:135-170, 247-272): `classes` holds per class its stacked expert tensors
    in LOCAL order and its expert map (int32 [num_experts]: global id -> local id, -1 for the other class's experts).
    topk_ids hold global ids; every id in [0, num_experts) must belong to exactly one class."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        raise ValueError("x must be a 2-D fp16/bf16 tensor")
    if not 1 <= len(classes) <= _lib.MAX_MOE_CLASSES:
        raise ValueError(f"1..{_lib.MAX_MOE_CLASSES} expert classes")
    T, H = x.shape
    arr = (_lib.Exl3MoeClass * len(classes))()
    I0 = None
    maps = []
    for c, (experts, emap) in enumerate(classes):
        E_c, I, K_gu, K_dn = _expert_stacks(experts, H, x.device)
        if I0 is not None and I != I0:
            raise ValueError("every class shares the intermediate width")
        I0 = I
        if emap.numel() != num_experts:
            raise ValueError(f"class {c}: expert map holds {emap.numel()} entries for {num_experts} experts")
        maps.append(_routing_ids(emap, x.device).reshape(-1))
        arr[c] = _lib.Exl3MoeClass(_lib.Exl3MoeWeights(*[experts[n].data_ptr() for n in MOE_TENSORS]),
                                   maps[-1].data_ptr(), E_c, K_gu, K_dn)
    ids, w = _routing(x, topk_ids, topk_weights)
    top_k = ids.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    _check_out(out, (T, H), x)
    lib = _lib.load()
    ws = workspace(x.device, lib.exl3_moe_classes_workspace_bytes(T, top_k, num_experts, H, I0, len(classes), arr),
                   "moe")
    _lib.check(lib.exl3_moe_forward_classes(x.contiguous().data_ptr(), int(x.dtype == torch.bfloat16), T, H,
                                            ids.data_ptr(), w.data_ptr(), top_k, num_experts, I0, arr, len(classes),
                                            int(codebook), out.data_ptr(), int(out.dtype == torch.bfloat16),
                                            ws.data_ptr(), ws.numel(), _stream(x.device)),
               "moe_forward_classes")
    return out


# ---- MoE per-launch stages: the launches the reference's unfused path runs after moe_align_block_size
# (cuda/src/sglang_exl3/kernels/marlin_moe.py:272-294: moe_had_in, moe_gemm for gate|up, moe_glu_had_in, moe_gemm for
# down, moe_combine), on the stored trellis stacks

def _routing_ids(topk_ids: torch.Tensor, device: torch.device) -> torch.Tensor:
    if topk_ids.dtype not in (torch.int32, torch.int64) or topk_ids.device != device:
        raise ValueError(f"topk_ids must be int32/int64 on {device}, got {topk_ids.dtype} on {topk_ids.device}")
    return topk_ids.to(torch.int32).contiguous()


def _ptr_array(tensors: list[torch.Tensor]):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def moe_align(topk_ids: torch.Tensor, num_experts: int, block: int, expert_map: torch.Tensor | None = None):
    """(sorted_ids, expert_ids, num_post_padded) in the layout of vLLM's moe_align_block_size for one block size
    (the reference's moe_align_decode, cuda/csrc/exl3_marlin_moe.cu:546-618): each expert's slots padded to a multiple
    of `block` with the sentinel topk_ids.numel(), the expert (or expert_map[e]) of every block, -1 past the end."""
    ids = _routing_ids(topk_ids, topk_ids.device).reshape(-1)
    slots = ids.numel()
    cap, max_blocks = moe_align_capacity(slots, num_experts, block)
    dev = ids.device
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    expert_ids = torch.empty(max_blocks, dtype=torch.int32, device=dev)
    post = torch.empty(1, dtype=torch.int32, device=dev)
    emap = None
    if expert_map is not None:
        if expert_map.numel() != num_experts:
            raise ValueError(f"expert_map holds {expert_map.numel()} entries for {num_experts} experts")
        emap = _routing_ids(expert_map, dev)
    _lib.check(_lib.load().exl3_moe_align(ids.data_ptr(), slots, int(num_experts), _ptr(emap), int(block),
                                          sorted_ids.data_ptr(), cap, expert_ids.data_ptr(), max_blocks,
                                          post.data_ptr(), _stream(dev)), "moe_align")
    return sorted_ids, expert_ids, post


def moe_align_classes(topk_ids: torch.Tensor, num_experts: int, expert_maps: list[torch.Tensor],
                      blocks: list[int]) -> list[tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """moe_align for every K class of a mixed layer in one launch (the reference's moe_align_decode,
    cuda/csrc/exl3_marlin_moe.cu:532-618): per class (sorted_ids, expert_ids, num_post_padded) as moe_align gives with
    that class's expert map and block size (local expert ids)."""
    n = len(expert_maps)
    if not 1 <= n <= _lib.MAX_MOE_CLASSES or len(blocks) != n:
        raise ValueError(f"1..{_lib.MAX_MOE_CLASSES} classes, one block size each")
    ids = _routing_ids(topk_ids, topk_ids.device).reshape(-1)
    slots, dev = ids.numel(), ids.device
    maps = []
    for emap in expert_maps:
        if emap.numel() != num_experts:
            raise ValueError(f"an expert map holds {emap.numel()} entries for {num_experts} experts")
        maps.append(_routing_ids(emap, dev).reshape(-1))
    out = []
    for b in blocks:
        cap, mb = moe_align_capacity(slots, num_experts, b)
        out.append((torch.empty(cap, dtype=torch.int32, device=dev), torch.empty(mb, dtype=torch.int32, device=dev),
                    torch.empty(1, dtype=torch.int32, device=dev)))
    P, I = ctypes.c_void_p, ctypes.c_int
    _lib.check(_lib.load().exl3_moe_align_classes(
        ids.data_ptr(), slots, int(num_experts), n, (P * n)(*[m.data_ptr() for m in maps]), (I * n)(*blocks),
        (P * n)(*[o[0].data_ptr() for o in out]), (I * n)(*[o[0].numel() for o in out]),
        (P * n)(*[o[1].data_ptr() for o in out]), (I * n)(*[o[1].numel() for o in out]),
        (P * n)(*[o[2].data_ptr() for o in out]), _stream(dev)), "moe_align_classes")
    return out


def moe_had_in(x: torch.Tensor, suh: list[torch.Tensor], topk_ids: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """xh [shards * slots, k] fp16: fp16(Had(fp16(x[token]) * suh_s[e])) per (shard, slot) (the reference's
    moe_had_in, cuda/csrc/exl3_marlin_moe.cu:416-448); suh: one [E, k] fp16 stack per shard (gate, up)."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        raise ValueError("x must be a 2-D fp16/bf16 tensor")
    T, k = x.shape
    ids = _routing_ids(topk_ids, x.device)
    if ids.dim() != 2 or ids.shape[0] != T:
        raise ValueError(f"topk_ids {tuple(topk_ids.shape)} must be [{T}, top_k]")
    if not 1 <= len(suh) <= 2:
        raise ValueError("one or two suh stacks")
    E = suh[0].shape[0]
    for t in suh:
        if t.dtype != torch.float16 or tuple(t.shape) != (E, k) or not t.is_contiguous() or t.device != x.device:
            raise ValueError(f"suh stacks must be contiguous fp16 [{E}, {k}] on {x.device}")
    slots = ids.numel()
    if out is None:
        out = torch.empty((len(suh) * slots, k), dtype=torch.float16, device=x.device)
    _check_out(out, (len(suh) * slots, k), x, (torch.float16,))
    _lib.check(_lib.load().exl3_moe_had_in(x.contiguous().data_ptr(), int(x.dtype == torch.bfloat16), T, k,
                                           ids.data_ptr(), ids.shape[1], E, _ptr_array(suh), len(suh),
                                           out.data_ptr(), _stream(x.device)), "moe_had_in")
    return out


def moe_gemm(a: torch.Tensor, trellis: list[torch.Tensor], svh: list[torch.Tensor] | None, sorted_ids: torch.Tensor,
             expert_ids: torch.Tensor, num_post_padded: torch.Tensor, block: int, codebook: int,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """The grouped expert GEMM over align blocks (the reference's moe_gemm, cuda/csrc/exl3_marlin_moe.cu:376-412):
    a fp16 [shards * rows, k] (rotated inputs), trellis one [E, k/16, n/16, 16K] stack per shard; returns c fp16
    [rows, shards * n], with the output transform fp16(Had(fp16(acc)) * svh) when svh stacks ([E, n]) are given."""
    if a.dtype != torch.float16 or a.dim() != 2 or not a.is_contiguous():
        raise ValueError("a must be a contiguous fp16 [shards * rows, k] tensor")
    shards = len(trellis)
    if shards not in (1, 2) or a.shape[0] % shards:
        raise ValueError(f"one or two trellis stacks; a has {a.shape[0]} rows")
    rows, k = a.shape[0] // shards, a.shape[1]
    t0 = trellis[0]
    if any(t.dtype != torch.int16 or t.dim() != 4 or t.shape != t0.shape or not t.is_contiguous()
           or t.device != a.device for t in trellis):
        raise ValueError("trellis stacks must be contiguous int16 [E, k/16, n/16, 16K] of one shape on a's device")
    E, n, K = t0.shape[0], t0.shape[2] * 16, bits_of(t0)
    if t0.shape[1] * 16 != k:
        raise ValueError(f"trellis input width {t0.shape[1] * 16} != {k}")
    if svh is not None:
        if len(svh) != shards or any(v.dtype != torch.float16 or tuple(v.shape) != (E, n) or not v.is_contiguous()
                                     or v.device != a.device for v in svh):
            raise ValueError(f"svh must be {shards} contiguous fp16 [{E}, {n}] stacks")
    for name, t in (("sorted_ids", sorted_ids), ("expert_ids", expert_ids), ("num_post_padded", num_post_padded)):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != a.device:
            raise ValueError(f"{name} must be a contiguous int32 tensor on {a.device}")
    max_blocks = expert_ids.numel()
    if max_blocks * block < sorted_ids.numel():
        raise ValueError(f"expert_ids ({max_blocks}) too short for {sorted_ids.numel()} sorted ids in blocks of {block}")
    if out is None:
        out = torch.empty((rows, shards * n), dtype=torch.float16, device=a.device)
    _check_out(out, (rows, shards * n), a, (torch.float16,))
    if rows == 0:
        return out
    lib = _lib.load()
    ws = workspace(a.device, lib.exl3_moe_gemm_workspace_bytes(rows, k, n, shards, max_blocks), "moe_stage")
    _lib.check(lib.exl3_moe_gemm(a.data_ptr(), rows, k, _ptr_array(trellis), None if svh is None else _ptr_array(svh),
                                 shards, n, sorted_ids.data_ptr(), expert_ids.data_ptr(), num_post_padded.data_ptr(),
                                 max_blocks, int(block), E, K, int(codebook), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                 _stream(a.device)), "moe_gemm")
    return out


def moe_glu_had_in(gu: torch.Tensor, suh_down: torch.Tensor, topk_ids: torch.Tensor, act: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(act, xd): act = fp16(silu(g) * u) and the rotated down inputs xd = fp16(Had(fp16(act * suh_down[e]))) per slot
    from gu fp16 [slots, 2 inter] (the reference's moe_glu_had_in, cuda/csrc/exl3_marlin_moe.cu:450-477)."""
    if gu.dtype != torch.float16 or gu.dim() != 2 or not gu.is_contiguous() or gu.shape[1] % 256:
        raise ValueError("gu must be a contiguous fp16 [slots, 2 inter] tensor")
    slots, inter = gu.shape[0], gu.shape[1] // 2
    ids = _routing_ids(topk_ids, gu.device).reshape(-1)
    if ids.numel() != slots:
        raise ValueError(f"topk_ids holds {ids.numel()} slots, gu {slots}")
    if suh_down.dtype != torch.float16 or suh_down.dim() != 2 or suh_down.shape[1] != inter \
            or not suh_down.is_contiguous() or suh_down.device != gu.device:
        raise ValueError(f"suh_down must be a contiguous fp16 [E, {inter}] stack")
    if act is None:
        act = torch.empty((slots, inter), dtype=torch.float16, device=gu.device)
    if out is None:
        out = torch.empty((slots, inter), dtype=torch.float16, device=gu.device)
    _check_out(act, (slots, inter), gu, (torch.float16,))
    _check_out(out, (slots, inter), gu, (torch.float16,))
    _lib.check(_lib.load().exl3_moe_glu_had_in(gu.data_ptr(), slots, inter, ids.data_ptr(), suh_down.shape[0],
                                               suh_down.data_ptr(), act.data_ptr(), out.data_ptr(),
                                               _stream(gu.device)), "moe_glu_had_in")
    return act, out


def moe_combine(yd: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, num_experts: int,
                out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """y [tokens, hidden] = sum_j w[t, j] * yd[t * top_k + j] in fp32, slot order, one rounding; slots with ids outside
    [0, num_experts) skipped (the reference's moe_combine, cuda/csrc/exl3_marlin_moe.cu:479-500)."""
    if yd.dtype != torch.float16 or yd.dim() != 2 or not yd.is_contiguous():
        raise ValueError("yd must be a contiguous fp16 [slots, hidden] tensor")
    ids = _routing_ids(topk_ids, yd.device)
    if ids.dim() != 2 or tuple(topk_weights.shape) != tuple(ids.shape) or ids.numel() != yd.shape[0]:
        raise ValueError(f"topk_ids {tuple(ids.shape)} / topk_weights {tuple(topk_weights.shape)} do not match "
                         f"{yd.shape[0]} rows")
    if topk_weights.device != yd.device:
        raise ValueError("topk_weights must be on yd's device")
    w = topk_weights.to(torch.float32).contiguous()
    T, top_k = ids.shape
    if out is None:
        out = torch.empty((T, yd.shape[1]), dtype=out_dtype, device=yd.device)
    _check_out(out, (T, yd.shape[1]), yd)
    _lib.check(_lib.load().exl3_moe_combine(yd.data_ptr(), w.data_ptr(), ids.data_ptr(), T, top_k, yd.shape[1],
                                            int(num_experts), out.data_ptr(), int(out.dtype == torch.bfloat16),
                                            _stream(yd.device)), "moe_combine")
    return out


def kv_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int,
                        sm_scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Single-token decode attention over a quantized paged KV cache (split-KV + log-sum-exp merge; the merge follows
    xpu/exl3xpu/fp8kv_prefill.py:85-117).  q fp16 [B, Hq, 128]; k_cache / v_cache int8 [P, Hkv, 16, 128] (bits=8)
    or uint8 [P, Hkv, 16, 64] (bits=4, packed nibbles); k_scale / v_scale fp16 [P, Hkv]; page_table int32
    [B, max_pages]; seq_lens int32 [B].  Returns fp16 [B, Hq, 128]."""
    if bits not in (4, 8):
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    if q.dtype != torch.float16 or q.dim() != 3:
        raise ValueError("q must be fp16 [B, Hq, D]")
    B, Hq, D = q.shape
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache / v_cache must have the same [P, Hkv, page, row] shape")
    P, Hkv, page, row = k_cache.shape
    if row != (D if bits == 8 else D // 2):
        raise ValueError(f"cache row of {row} bytes does not hold {D} {bits}-bit codes")
    if k_cache.element_size() != 1 or v_cache.element_size() != 1:
        raise ValueError("caches must hold 1-byte codes (int8 / uint8)")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != torch.float16 or tuple(t.shape) != (P, Hkv):
            raise ValueError(f"{name} must be fp16 [{P}, {Hkv}]")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError("page_table must be int32 [B, max_pages]")
    if seq_lens.dtype != torch.int32 or tuple(seq_lens.shape) != (B,):
        raise ValueError("seq_lens must be int32 [B]")
    tensors = (q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens)
    if not all(t.is_cuda and t.is_contiguous() and t.device == q.device for t in tensors):
        raise ValueError("all inputs must be contiguous CUDA tensors on one device")
    if sm_scale is None:
        sm_scale = D ** -0.5
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float16, device=q.device)
    _check_out(out, (B, Hq, D), q, (torch.float16,))
    lib = _lib.load()
    max_pages = page_table.shape[1]
    ws = workspace(q.device, lib.exl3_kv_decode_workspace_bytes(B, Hq, Hkv, max_pages), "kv")
    _lib.check(lib.exl3_kv_decode_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                                            v_scale.data_ptr(), P, page_table.data_ptr(), max_pages,
                                            seq_lens.data_ptr(), B, Hq, Hkv, D, page, int(bits), float(sm_scale),
                                            out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(q.device)),
               "kv_decode_attention")
    return out


# ---- Around the quantized-KV attention: what a decode or speculative step does between its linears and the cache.  The
# reference has no counterpart of these (its engines bring them).  Their workspaces come from torch's allocator on the
# current stream, call by call: calls on several streams and captured graphs never share one.  A caller's own `workspace`
# saves that allocation (and its `out`, where there is one, the results'; verify_drafts makes its own); calls that share it
# must then be ordered.

# The checks are written for their cost: the library call of 23 arguments and its launch take 3.7 us, each attribute read of
# a tensor 0.06 to 0.09, an allocation 1.5 (new_empty) to 1.7.

_HEAD_DIM = 128
_HALVES = (torch.float16, torch.bfloat16)
_FP16 = (torch.float16,)
_WEIGHT_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_INTS = (torch.int32, torch.int64)


def _token_stride(t: torch.Tensor, name: str, dims: int, dtypes=_HALVES) -> int:
    """Elements from one token's heads to the next's in t [..., heads, 128] (`dims` dimensions): columns of a wider row
    are fine, a token's heads are contiguous."""
    shape, stride = t.shape, t.stride()
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if len(shape) != dims or shape[-1] != _HEAD_DIM:
        raise ValueError(f"{name} must be a {dims}-D tensor [..., heads, {_HEAD_DIM}], got {tuple(shape)}")
    if stride[-1] != 1 or (stride[-2] != _HEAD_DIM and shape[-2] > 1):
        raise ValueError(f"{name}: a token's heads must be contiguous, got strides {stride}")
    if dims == 3:
        return stride[0] if shape[0] > 1 else shape[1] * _HEAD_DIM
    B, n, heads, _ = shape
    if n == 1:
        return stride[0] if B > 1 else heads * _HEAD_DIM
    if B > 1 and stride[0] != n * stride[1]:
        raise ValueError(f"{name}: the sequences' tokens must lie at one stride, got strides {stride}")
    return stride[1]


def _check_int32(t: torch.Tensor | None, name: str, shape: tuple) -> None:
    if t is not None and (t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int) -> tuple[int, int, int, int]:
    """Checks a paged cache as kv_decode_attention takes it; returns (pages, kv heads, sequences, table width)."""
    if bits != 8 and bits != 4:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or shape[2] != 16 or shape[3] != 16 * bits:
        raise ValueError(f"k_cache / v_cache must both be [P, Hkv, 16, {16 * bits}] at {bits} bits, got "
                         f"{tuple(shape)} / {tuple(v_cache.shape)}")
    if k_cache.element_size() != 1 or v_cache.element_size() != 1:
        raise ValueError("caches must hold 1-byte codes (int8 / uint8)")
    P, Hkv = shape[0], shape[1]
    if k_scale.dtype != torch.float16 or k_scale.shape != (P, Hkv):
        raise ValueError(f"k_scale must be fp16 [{P}, {Hkv}]")
    if v_scale.dtype != torch.float16 or v_scale.shape != (P, Hkv):
        raise ValueError(f"v_scale must be fp16 [{P}, {Hkv}]")
    table = page_table.shape
    if page_table.dtype != torch.int32 or len(table) != 2:
        raise ValueError("page_table must be int32 [B, max_pages]")
    B, max_pages = table
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,):
        raise ValueError(f"seq_lens must be int32 [{B}]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
            and page_table.is_contiguous() and seq_lens.is_contiguous()):
        raise ValueError("caches, scales, page table and lengths must be contiguous")
    return P, Hkv, B, max_pages


def _check_apart(out: torch.Tensor, *inputs) -> None:
    """An output (or a workspace) that other workgroups' inputs lie in would be read and written in any order."""
    start = out.data_ptr()
    for t in inputs:
        if t is not None and t.numel() and out.numel():
            at = t.data_ptr()
            span = t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            if at < start + out.nbytes and start < at + span:
                raise ValueError("an output overlaps another tensor of the call")


def _cuda_index(first: torch.Tensor, *others) -> int:
    """The index of the device that all tensors are on (None: no tensor)."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"all tensors must be on one device, got {t.device} and {first.device}")
    if index < 0:
        raise ValueError(f"Expected a cuda device, but got: {first.device}")
    return index


def _current(index: int) -> bool:
    return torch._C._cuda_getDevice() == index


def _call_workspace(workspace: torch.Tensor | None, nbytes: int, like: torch.Tensor) -> torch.Tensor:
    if workspace is None:
        return like.new_empty(max(nbytes, 16), dtype=torch.uint8)
    if not workspace.is_contiguous() or workspace.device != like.device:
        raise ValueError(f"workspace must be a contiguous tensor on {like.device}")
    return workspace


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 cos_sin: torch.Tensor | None, positions: torch.Tensor | None, eps: float = 1e-6,
                 interleaved: bool = False, out_dtype: torch.dtype | None = None,
                 out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The norm of every query and key head and its rotation by the token's position, in one launch.
    q fp16|bf16 [T, Hq, 128], k [T, Hkv, 128], columns of the fused q/k/v linear's output or tensors of their own;
    q_weight, k_weight fp16|bf16|fp32 [128] (both None: no norm); cos_sin fp32 [max_pos, rotary] holds the cosines and then
    the sines of every position (rotary a multiple of 16 up to 128; None: no rotation), positions int32|int64 [T] (clamped
    into the table).  Pairs are (i, i + rotary / 2), or (2i, 2i + 1) when `interleaved`.  fp32 inside; returns (q, k)
    contiguous in `out_dtype` (q's by default; fp16 for the attention over the cache), in `out` if given (which may be q
    and k themselves where those are contiguous and of one type)."""
    ld_q, ld_k = _token_stride(q, "q", 3), _token_stride(k, "k", 3)
    T, Hq, _ = q.shape
    Tk, Hkv, _ = k.shape
    dtype = q.dtype
    if Tk != T or k.dtype != dtype:
        raise ValueError(f"k must hold {T} tokens in {dtype}, got {Tk} in {k.dtype}")
    w_type = max_pos = rotary = wide = 0
    wq = wk = cs = pos = None
    if q_weight is not None and k_weight is not None:
        w_dtype = q_weight.dtype
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w.dtype != w_dtype or w_dtype not in _WEIGHT_TYPE or w.shape != (_HEAD_DIM,) or not w.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [{_HEAD_DIM}] tensor, both of one type (fp16, bf16, fp32)")
        w_type, wq, wk = _WEIGHT_TYPE[w_dtype], q_weight.data_ptr(), k_weight.data_ptr()
    elif q_weight is not None or k_weight is not None:
        raise ValueError("both weights or neither")
    elif cos_sin is None:
        raise ValueError("neither weights nor a rotation table")
    if cos_sin is not None:
        shape = cos_sin.shape
        if cos_sin.dtype != torch.float32 or len(shape) != 2 or not cos_sin.is_contiguous():
            raise ValueError("cos_sin must be a contiguous fp32 [max_pos, rotary] tensor")
        if positions is None or positions.dtype not in _INTS or positions.shape != (T,) or not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int32/int64 [{T}] tensor")
        max_pos, rotary = shape
        if max_pos < 1 or rotary % 16 or not 16 <= rotary <= _HEAD_DIM:
            raise ValueError(f"cos_sin {tuple(shape)}: rotary must be a multiple of 16 up to {_HEAD_DIM}")
        cs, pos, wide = cos_sin.data_ptr(), positions.data_ptr(), int(positions.dtype == torch.int64)
    if out is None:
        out_dtype = out_dtype or dtype
        if out_dtype not in _HALVES:
            raise ValueError(f"out_dtype must be fp16 or bf16, got {out_dtype}")
    else:
        q_out, k_out = out
        _check_out(q_out, (T, Hq, _HEAD_DIM), q)
        _check_out(k_out, (T, Hkv, _HEAD_DIM), q)
        if q_out.dtype != k_out.dtype or out_dtype not in (None, q_out.dtype):
            raise ValueError(f"outputs of one type, got {q_out.dtype}, {k_out.dtype}")
        out_dtype = q_out.dtype
        for x, o in ((q, q_out), (k, k_out)):
            if x.data_ptr() != o.data_ptr():
                _check_apart(o, x)
            elif x.dtype != o.dtype or not x.is_contiguous():
                raise ValueError("an output may be its input only where both are contiguous and of one type")
        rest = (q_weight, k_weight, cos_sin, positions if cos_sin is not None else None)
        _check_apart(q_out, k, k_out, *rest)
        _check_apart(k_out, q, *rest)
    index = _cuda_index(q, k, q_weight, k_weight, cos_sin, positions if cos_sin is not None else None)
    if not _current(index):
        with torch.cuda.device(index):
            return qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, out_dtype, out)
    if out is None:
        q_out = q.new_empty((T, Hq, _HEAD_DIM), dtype=out_dtype)
        k_out = q.new_empty((T, Hkv, _HEAD_DIM), dtype=out_dtype)
    _lib.check(_lib.load().exl3_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), dtype == torch.bfloat16, ld_q, ld_k, T, Hq, Hkv, _HEAD_DIM, wq, wk, w_type, eps, cs,
        max_pos, rotary, interleaved, pos, wide, q_out.data_ptr(), k_out.data_ptr(), out_dtype == torch.bfloat16,
        torch._C._cuda_getCurrentRawStream(index)), "qk_norm_rope")
    return q_out, k_out


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int,
              row_start: torch.Tensor | None = None, max_new: int | None = None, select: torch.Tensor | None = None,
              counts: torch.Tensor | None = None) -> None:
    """Quantizes new keys and values into the paged cache (the layout of kv_decode_attention), at positions seq_lens[b],
    seq_lens[b] + 1, ... of sequence b; seq_lens (the lengths before the call) are not changed.  k, v fp16|bf16, columns of
    a wider row allowed:
      [B, n, Hkv, 128]     n rows a sequence (with `counts` int32 [B]: the first counts[b] of them);
      [B, Hkv, 128]        one a sequence;
      [rows, Hkv, 128]     with row_start int32 [B + 1], ascending: rows row_start[b] .. row_start[b + 1] - 1 are sequence b's
                           (`max_new`: the most a sequence has, if known on the host; it sizes the launch).
    No sequence gets more than `max_new` tokens, where it is given.
    select int32 [B, S]: token j of sequence b is its row select[b, j] (the accepted nodes of verify_drafts, with its
    `counts`).  A page's scale covers its new tokens and what it held; older codes are rounded anew where it grows.  Tokens
    past the table and pages outside the cache are not written; no two sequences may append to one page."""
    P, Hkv, B, max_pages = _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits)
    shape = k.shape
    dims = len(shape)
    if dims not in (3, 4) or (dims == 4 and row_start is not None):
        raise ValueError("k must be [B, n, Hkv, 128], [B, Hkv, 128], or [rows, Hkv, 128] with row_start")
    ld_k, ld_v = _token_stride(k, "k", dims), _token_stride(v, "v", dims)
    dtype = k.dtype
    if v.shape != shape or v.dtype != dtype or shape[-2] != Hkv:
        raise ValueError(f"k {tuple(shape)} {dtype} and v {tuple(v.shape)} {v.dtype} must be alike, of {Hkv} heads")
    rows = shape[0] * shape[1] if dims == 4 else shape[0]
    per_seq = 0
    starts = picks = limits = None
    if row_start is None:
        if shape[0] != B:
            raise ValueError(f"k holds {shape[0]} sequences, the page table {B}")
        per_seq = shape[1] if dims == 4 else 1
    else:
        _check_int32(row_start, "row_start", (B + 1,))
        starts = row_start.data_ptr()
    if counts is not None:
        _check_int32(counts, "counts", (B,))
        limits = counts.data_ptr()
    if select is not None:
        if select.dim() != 2:
            raise ValueError(f"select must be int32 [{B}, S]")
        if max_new is not None and max_new < select.shape[1]:
            raise ValueError(f"max_new = {max_new}, but select names up to {select.shape[1]} tokens (limit them by counts)")
        max_new = select.shape[1]
        _check_int32(select, "select", (B, max_new))
        picks = select.data_ptr()
    else:
        most = rows if row_start is not None else per_seq
        max_new = most if max_new is None else min(max_new, most)
    if max_new < 0:
        raise ValueError(f"max_new = {max_new}")
    index = _cuda_index(k, v, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, row_start, select, counts)
    if not _current(index):
        with torch.cuda.device(index):
            return kv_append(k, v, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits, row_start, max_new,
                             select, counts)
    _lib.check(_lib.load().exl3_kv_append(
        k.data_ptr(), v.data_ptr(), dtype == torch.bfloat16, ld_k, ld_v, rows, starts, per_seq, picks, limits, max_new,
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, page_table.data_ptr(), max_pages,
        seq_lens.data_ptr(), B, Hkv, _HEAD_DIM, 16, bits, torch._C._cuda_getCurrentRawStream(index)), "kv_append")


def kv_gather(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
              page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int, row_start: torch.Tensor, rows: int,
              starts: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
              out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads the paged cache back: (k, v) fp16|bf16 [rows, Hkv, 128] whose row row_start[b] + i is token starts[b] + i of
    sequence b, for the rows below row_start[b + 1] (int32 [B + 1], ascending) and the tokens below seq_lens[b]; starts int32
    [B] (None: 0).  Other rows are left as they were (in tensors made here: uninitialised).  Page ids outside the cache are
    clamped."""
    P, Hkv, B, max_pages = _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits)
    _check_int32(row_start, "row_start", (B + 1,))
    first = None
    if starts is not None:
        _check_int32(starts, "starts", (B,))
        first = starts.data_ptr()
    shape = (rows, Hkv, _HEAD_DIM)
    if out is None:
        if dtype not in _HALVES or rows < 0:
            raise ValueError(f"rows = {rows}; dtype must be fp16 or bf16, got {dtype}")
    else:
        k_out, v_out = out
        dtype = k_out.dtype
        _check_out(k_out, shape, k_cache)
        _check_out(v_out, shape, k_cache, (dtype,))
        read = (k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, row_start, starts)
        _check_apart(k_out, v_out, *read)
        _check_apart(v_out, *read)
    index = _cuda_index(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, row_start, starts)
    if not _current(index):
        with torch.cuda.device(index):
            return kv_gather(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits, row_start, rows, starts,
                             dtype, out)
    if out is None:
        k_out = k_scale.new_empty(shape, dtype=dtype)
        v_out = k_scale.new_empty(shape, dtype=dtype)
    _lib.check(_lib.load().exl3_kv_gather(
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, page_table.data_ptr(),
        max_pages, seq_lens.data_ptr(), first, row_start.data_ptr(), B, rows, Hkv, _HEAD_DIM, 16, bits, k_out.data_ptr(),
        v_out.data_ptr(), dtype == torch.bfloat16, torch._C._cuda_getCurrentRawStream(index)), "kv_gather")
    return k_out, v_out


def kv_tree_workspace_bytes(batch: int, nodes: int, num_q_heads: int, num_kv_heads: int, max_pages: int) -> int:
    """Bytes of a `workspace` for kv_tree_attention at this shape."""
    return _lib.load().exl3_kv_tree_workspace_bytes(batch, nodes, num_q_heads, num_kv_heads, max_pages)


def kv_tree_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, tree_mask: torch.Tensor | None,
                      k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                      page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int, sm_scale: float | None = None,
                      num_nodes: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's drafted tokens over the paged quantized cache and over each other.  q fp16
    [B, N, Hq, 128], k_new / v_new fp16 [B, N, Hkv, 128] (N <= 64; columns of the fused linear's output allowed): every node
    sees the seq_lens[b] cached tokens, and node i those nodes j of its sequence with bit j of tree_mask[b, i] set (int64
    [B, N]; its own too, as a rule; None: nodes 0 .. i, a chain or a prompt's chunk).  num_nodes int32 [B]: the nodes of a
    sequence from there on are neither read nor written.  A node that sees nothing gives zeros.  Cache as
    kv_decode_attention; returns fp16 [B, N, Hq, 128]."""
    P, Hkv, B, max_pages = _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits)
    ld_q, ld_k, ld_v = (_token_stride(q, "q", 4, _FP16), _token_stride(k_new, "k_new", 4, _FP16),
                        _token_stride(v_new, "v_new", 4, _FP16))
    Bq, N, Hq, _ = q.shape
    if Bq != B or k_new.shape != (B, N, Hkv, _HEAD_DIM) or v_new.shape != k_new.shape:
        raise ValueError(f"q {tuple(q.shape)}, k_new {tuple(k_new.shape)} and v_new {tuple(v_new.shape)} do not match "
                         f"{B} sequences and {Hkv} kv heads")
    if not 1 <= N <= 64 or Hq % Hkv or not 1 <= Hq // Hkv <= 16:
        raise ValueError(f"1 to 64 nodes and 1 to 16 query heads per kv head, got {N} nodes, heads {Hq} / {Hkv}")
    mask = live = None
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.shape != (B, N) or not tree_mask.is_contiguous():
            raise ValueError(f"tree_mask must be a contiguous int64 [{B}, {N}] tensor")
        mask = tree_mask.data_ptr()
    if num_nodes is not None:
        _check_int32(num_nodes, "num_nodes", (B,))
        live = num_nodes.data_ptr()
    if out is not None:
        _check_out(out, (B, N, Hq, _HEAD_DIM), q, _FP16)
        _check_apart(out, q, k_new, v_new, tree_mask, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, num_nodes)
    if workspace is not None:
        _check_apart(workspace, out, q, k_new, v_new, tree_mask, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens,
                     num_nodes)
    index = _cuda_index(q, k_new, v_new, tree_mask, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, num_nodes)
    if sm_scale is None:
        sm_scale = _HEAD_DIM ** -0.5
    if not _current(index):
        with torch.cuda.device(index):
            return kv_tree_attention(q, k_new, v_new, tree_mask, k_cache, v_cache, k_scale, v_scale, page_table,
                                     seq_lens, bits, sm_scale, num_nodes, out, workspace)
    if out is None:
        out = q.new_empty((B, N, Hq, _HEAD_DIM))
    lib = _lib.load()
    ws = _call_workspace(workspace, lib.exl3_kv_tree_workspace_bytes(B, N, Hq, Hkv, max_pages), q)
    _lib.check(lib.exl3_kv_tree_attention(
        q.data_ptr(), ld_q, k_new.data_ptr(), v_new.data_ptr(), ld_k, ld_v, mask, N, live, k_cache.data_ptr(),
        v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, page_table.data_ptr(), max_pages,
        seq_lens.data_ptr(), B, Hq, Hkv, _HEAD_DIM, 16, bits, sm_scale, out.data_ptr(), ws.data_ptr(), ws.nbytes,
        torch._C._cuda_getCurrentRawStream(index)), "kv_tree_attention")
    return out


def verify_workspace_bytes(batch: int, vocab: int) -> int:
    """Bytes of a `workspace` for verify_drafts at this shape."""
    return _lib.load().exl3_verify_workspace_bytes(batch, vocab)


def _narrow(t: torch.Tensor, end: int) -> torch.Tensor:
    """int32 values; what lies outside [0, end) stays outside."""
    if t.dtype == torch.int64:
        t = t.clamp(-1, end).to(torch.int32)
    return t.contiguous()


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, uniform: torch.Tensor,
                  parents: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None,
                  num_nodes: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stay, and the token after them, so that every emitted token is distributed as the target's.
    Node 0 of a sequence is its last committed token, nodes 1 .. N - 1 are drafts (N <= 64).  target_probs fp32 [B, N, V]:
    row i after node i; tokens int32|int64 [B, N]; uniform fp32 [B, N] in [0, 1): u[b, i] decides node i, u[b, 0] draws the
    next token; parents int32|int64 [B, N], a node's parent before it (None: a chain); num_nodes int32 [B] (None: N each).
      draft_probs fp32 [B, N, V] (chains): row i is what node i + 1 was drawn from; accepted while u q(t) < p(t), the next
        token from max(p - q, 0) after a refusal;
      None: candidates however chosen; brothers in order, accepted when u m < p(t) with m = 1 less their refused brothers'
        p, refused tokens struck from p.
    Returns (accepted_nodes [B, N]: 0, then the accepted drafts; counts [B]: how many of them, the root among them;
    out_tokens [B, N]: the accepted drafts' tokens, then the next one), int32, -1 past counts[b].  accepted_nodes and counts
    are what kv_append takes as `select` and `counts`."""
    shape = target_probs.shape
    if target_probs.dtype != torch.float32 or len(shape) != 3 or not target_probs.is_contiguous():
        raise ValueError(f"target_probs must be a contiguous fp32 [B, N, V] tensor, got {target_probs.dtype} "
                         f"{tuple(shape)}")
    B, N, V = shape
    if not 1 <= N <= 64 or V < 1:
        raise ValueError(f"1 to 64 nodes and at least one token, got {N} nodes, {V} tokens")
    for name, t in (("tokens", tokens), ("parents", parents)):
        if t is not None and (t.dtype not in _INTS or t.shape != (B, N)):
            raise ValueError(f"{name} must be int32/int64 [{B}, {N}], got {t.dtype} {tuple(t.shape)}")
    if uniform.dtype != torch.float32 or uniform.shape != (B, N) or not uniform.is_contiguous():
        raise ValueError(f"uniform must be a contiguous fp32 [{B}, {N}] tensor")
    q = up = live = None
    if draft_probs is not None:
        if parents is not None:
            raise ValueError("the draft's probabilities come with a chain (parents = None)")
        if draft_probs.dtype != torch.float32 or draft_probs.shape != shape or not draft_probs.is_contiguous():
            raise ValueError(f"draft_probs must be a contiguous fp32 [{B}, {N}, {V}] tensor")
        q = draft_probs.data_ptr()
    if num_nodes is not None:
        _check_int32(num_nodes, "num_nodes", (B,))
        live = num_nodes.data_ptr()
    if workspace is not None:
        _check_apart(workspace, target_probs, tokens, uniform, parents, draft_probs, num_nodes)
    index = _cuda_index(target_probs, tokens, uniform, parents, draft_probs, num_nodes)
    if not _current(index):
        with torch.cuda.device(index):
            return verify_drafts(target_probs, tokens, uniform, parents, draft_probs, num_nodes, workspace)
    tokens = _narrow(tokens, V)
    if parents is not None:
        parents = _narrow(parents, N)
        up = parents.data_ptr()
    accepted = tokens.new_empty((B, N))
    out_tokens = tokens.new_empty((B, N))
    counts = tokens.new_empty(B)
    lib = _lib.load()
    ws = _call_workspace(workspace, lib.exl3_verify_workspace_bytes(B, V), tokens)
    _lib.check(lib.exl3_verify_drafts(
        target_probs.data_ptr(), q, tokens.data_ptr(), up, uniform.data_ptr(), live, B, N, V, accepted.data_ptr(),
        counts.data_ptr(), out_tokens.data_ptr(), ws.data_ptr(), ws.nbytes,
        torch._C._cuda_getCurrentRawStream(index)), "verify_drafts")
    return accepted, counts, out_tokens


# ---- Around the attention and at the ends of a serving step: pages and rows from the requests' lengths, the step between two
# blocks, attention over chosen pages, sampling.  Workspaces as above.

class StepPlan(NamedTuple):
    """What kv_step_plan returns, int32 (slots int64): of the sequences row_start [B + 1], counts [B], lens_after [B]; of the
    step's rows positions, row_lens, row_seq and slots [rows]."""
    row_start: torch.Tensor
    counts: torch.Tensor
    lens_after: torch.Tensor
    positions: torch.Tensor
    row_lens: torch.Tensor
    row_seq: torch.Tensor
    slots: torch.Tensor


def kv_step_plan(page_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                 free_state: torch.Tensor, rows: int, state_out: torch.Tensor | None = None) -> StepPlan:
    """The pages, rows and slots of a step from the requests' lengths, without the host knowing them.  Sequence b holds
    seq_lens[b] tokens and asks for new_lens[b] more (int32 [B]), or, below 0, gives its last -new_lens[b] ones up.  free_pages
    int32 is a ring of free page ids, free_state int32 [2] the place of its first live entry and how many are live: pages are
    taken from its beginning in order of b and written into page_table int32 [B, max_pages]; pages given up go to its end;
    state_out (None: free_state itself) gets its state after the step.  The ring is to have a place for every page that is ever
    live in it: given-up pages past its places are left out.  A sequence gets all of its tokens or none: none when its
    table row is too short, its rows pass `rows`, or the pages asked for so far are more than there are.
    Returns, for the step's `rows` rows (new token i of b is row row_start[b] + i): row_start (kv_append's), counts (the tokens
    got; kv_append's), lens_after, positions (qk_norm_rope's), row_lens and row_seq (kv_select_pages' and
    kv_sparse_attention's seq_lens and row_seq), slots (page * 16 + place).  Rows of refused sequences and behind the last one
    have -1, 0, -1 and -1."""
    shape = page_table.shape
    if page_table.dtype != torch.int32 or len(shape) != 2 or not page_table.is_contiguous():
        raise ValueError(f"page_table must be a contiguous int32 [B, max_pages] tensor, got {page_table.dtype} {tuple(shape)}")
    B, max_pages = shape
    _check_int32(seq_lens, "seq_lens", (B,))
    _check_int32(new_lens, "new_lens", (B,))
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise ValueError(f"free_pages must be a contiguous int32 [P] tensor, got {free_pages.dtype} {tuple(free_pages.shape)}")
    _check_int32(free_state, "free_state", (2,))
    if state_out is None:
        state_out = free_state
    else:
        _check_int32(state_out, "state_out", (2,))
    if rows < 0:
        raise ValueError(f"rows = {rows}")
    index = _cuda_index(page_table, seq_lens, new_lens, free_pages, free_state, state_out)
    if not _current(index):
        with torch.cuda.device(index):
            return kv_step_plan(page_table, seq_lens, new_lens, free_pages, free_state, rows, state_out)
    # one allocation, the workspace at its end
    buf = page_table.new_empty(5 * rows + 4 * B + 5)
    at_slots = buf.data_ptr()
    at_start = at_slots + 8 * rows
    at_counts = at_start + 4 * B + 4
    at_after = at_counts + 4 * B
    at_pos = at_after + 4 * B
    at_lens = at_pos + 4 * rows
    at_seq = at_lens + 4 * rows
    _lib.check(_lib.load().exl3_kv_step_plan(
        page_table.data_ptr(), max_pages, seq_lens.data_ptr(), new_lens.data_ptr(), B, 16, free_pages.data_ptr(),
        free_pages.numel(), free_state.data_ptr(), state_out.data_ptr(), rows, at_start, at_counts, at_after, at_pos, at_lens,
        at_seq, at_slots, at_seq + 4 * rows, 4 * (B + 4), torch._C._cuda_getCurrentRawStream(index)), "kv_step_plan")
    slots, row_start, counts, after, positions, row_lens, row_seq, _ = buf.split_with_sizes(
        (2 * rows, B + 1, B, B, rows, rows, rows, B + 4))
    if B == 0:  # (the library writes nothing)
        row_start.zero_()
        if state_out is not free_state:
            state_out.copy_(free_state)
    return StepPlan(row_start, counts, after, positions, row_lens, row_seq, slots.view(torch.int64))


def _row_stride(t: torch.Tensor, name: str, shape: tuple, dtypes) -> int:
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: a row's values must be contiguous, got strides {stride}")
    return stride[0] if shape[0] > 1 else shape[1]


def add_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float = 1e-6,
             post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_sigmoid: bool = False,
             scale: float = 1.0, unit_offset: bool = False,
             out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None
             ) -> tuple[torch.Tensor | None, torch.Tensor]:
    """From one block to the next in one launch: u = x, a block's output fp16|bf16 [T, dim] (with post_weight its RMS norm);
    h = residual + scale * gate * u; y = RMS norm of h by `weight`.  Returns (y, h): y in x's type, h in the residual's (fp16,
    bf16 or fp32; x's where there is none).  weight None: y is None (after the last block of a part).  gate [dim], [T, 1] or
    [T, dim] (taken through a sigmoid with gate_sigmoid); weights and gate fp16|bf16|fp32, weights of one type, as 1 + w with
    unit_offset.  fp32 inside, y from the h before its rounding.  out: (y, h) to write to; h may be the residual itself where
    that is contiguous."""
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2:
        raise ValueError(f"x must be [T, dim], got {tuple(shape)}")
    T, dim = shape
    ld_x = _row_stride(x, "x", shape, _HALVES)
    r_dtype, ld_r = dtype, dim
    if residual is not None:
        ld_r = _row_stride(residual, "residual", shape, _WEIGHT_TYPE)
        r_dtype = residual.dtype
    w_type = g_type = kind = ld_g = 0
    w_dtype = None
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is not None:
            w_dtype = w_dtype or w.dtype
            if w.dtype != w_dtype or w_dtype not in _WEIGHT_TYPE or w.shape != (dim,) or not w.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [{dim}] tensor, both weights of one type (fp16, bf16, fp32)")
            w_type = _WEIGHT_TYPE[w_dtype]
    if gate is not None:
        if gate.dtype not in _WEIGHT_TYPE:
            raise ValueError(f"gate must be fp16, bf16 or fp32, got {gate.dtype}")
        g_type, g_shape = _WEIGHT_TYPE[gate.dtype], gate.shape
        if g_shape == (dim,) and gate.is_contiguous():
            kind = 1
        elif g_shape == shape and dim > 1:
            kind, ld_g = 3, _row_stride(gate, "gate", shape, _WEIGHT_TYPE)
        elif g_shape == (T, 1):
            kind, ld_g = 2, gate.stride(0) if T > 1 else 1
        else:
            raise ValueError(f"gate must be a contiguous [{dim}] tensor, [{T}, 1] or [{T}, {dim}], got {tuple(g_shape)}")
        if kind == 2 and ld_g < 1:
            raise ValueError(f"gate: strides {gate.stride()}")
    y = h = None
    if out is not None:
        y, h = out
        if (y is None) != (weight is None):
            raise ValueError("out[0] comes with a weight")
        if y is not None:
            _check_out(y, shape, x, (dtype,))
        if h is not None:
            _check_out(h, shape, x, (r_dtype,))
    index = _cuda_index(x, residual, weight, post_weight, gate)
    if not _current(index):
        with torch.cuda.device(index):
            return add_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, unit_offset, out)
    if y is None and weight is not None:
        y = x.new_empty(shape)
    if h is None:
        h = x.new_empty(shape, dtype=r_dtype)
    _lib.check(_lib.load().exl3_add_norm(
        x.data_ptr(), dtype == torch.bfloat16, ld_x, _ptr(residual), _WEIGHT_TYPE[r_dtype], ld_r, _ptr(weight),
        _ptr(post_weight), w_type, unit_offset, _ptr(gate), g_type, kind, ld_g, gate_sigmoid, scale, eps, T, dim, _ptr(y),
        h.data_ptr(), torch._C._cuda_getCurrentRawStream(index)), "add_norm")
    return y, h


def kv_page_bounds(k_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int, bounds: torch.Tensor,
                   first: torch.Tensor | None = None, max_new: int | None = None) -> None:
    """Makes anew, in `bounds` ([P, Hkv, 2, 16 * bits], 1-byte like k_cache and packed like its rows), the largest and the
    smallest key code of every channel of the pages that hold tokens first[b] .. seq_lens[b] - 1 of sequence b (int32 [B]; first
    None: 0), of which the last `max_new` at most, if given (it sizes the launch).  After kv_append: first = the lengths before
    it, seq_lens = those after (kv_step_plan's lens_after).  Bounds are codes: they go with the page's k_scale."""
    if bits != 8 and bits != 4:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    shape = k_cache.shape
    if len(shape) != 4 or shape[2] != 16 or shape[3] != 16 * bits or k_cache.element_size() != 1:
        raise ValueError(f"k_cache must be 1-byte [P, Hkv, 16, {16 * bits}] at {bits} bits, got {tuple(shape)}")
    P, Hkv = shape[0], shape[1]
    if bounds.shape != (P, Hkv, 2, 16 * bits) or bounds.element_size() != 1:
        raise ValueError(f"bounds must be 1-byte [{P}, {Hkv}, 2, {16 * bits}], got {bounds.dtype} {tuple(bounds.shape)}")
    table = page_table.shape
    if page_table.dtype != torch.int32 or len(table) != 2:
        raise ValueError("page_table must be int32 [B, max_pages]")
    B, max_pages = table
    if not (k_cache.is_contiguous() and bounds.is_contiguous() and page_table.is_contiguous()):
        raise ValueError("the cache, the bounds and the page table must be contiguous")
    _check_int32(seq_lens, "seq_lens", (B,))
    _check_int32(first, "first", (B,))
    max_new = 16 * max_pages if max_new is None else min(max_new, 16 * max_pages)
    if max_new < 0:
        raise ValueError(f"max_new = {max_new}")
    index = _cuda_index(k_cache, page_table, seq_lens, bounds, first)
    if not _current(index):
        with torch.cuda.device(index):
            return kv_page_bounds(k_cache, page_table, seq_lens, bits, bounds, first, max_new)
    _lib.check(_lib.load().exl3_kv_page_bounds(
        k_cache.data_ptr(), P, page_table.data_ptr(), max_pages, seq_lens.data_ptr(), _ptr(first), max_new, B, Hkv, _HEAD_DIM,
        16, bits, bounds.data_ptr(), torch._C._cuda_getCurrentRawStream(index)), "kv_page_bounds")


def _check_rows(q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, row_seq: torch.Tensor | None,
                Hkv: int) -> tuple[int, int, int, int, int]:
    """Query rows of a paged cache; returns (row stride, rows, query heads, sequences, table width)."""
    ld_q = _token_stride(q, "q", 3, _FP16)
    R, Hq, _ = q.shape
    if Hkv < 1 or Hq % Hkv or not 1 <= Hq // Hkv <= 16:
        raise ValueError(f"1 to 16 query heads per kv head, got heads {Hq} / {Hkv}")
    table = page_table.shape
    if page_table.dtype != torch.int32 or len(table) != 2 or not page_table.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 [B, max_pages] tensor")
    _check_int32(seq_lens, "seq_lens", (R,))
    _check_int32(row_seq, "row_seq", (R,))
    if row_seq is None and R != table[0]:
        raise ValueError(f"{R} rows of {table[0]} sequences need row_seq")
    return ld_q, R, Hq, table[0], table[1]


def kv_select_workspace_bytes(rows: int, num_kv_heads: int, max_pages: int) -> int:
    """Bytes of a `workspace` for kv_select_pages of up to `rows` rows."""
    return _lib.load().exl3_kv_select_workspace_bytes(rows, num_kv_heads, max_pages)


def kv_select_pages(q: torch.Tensor, bounds: torch.Tensor, k_scale: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, bits: int, top: int, first: int = 1, last: int = 2,
                    row_seq: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The pages that each query row is to read: int32 [R, Hkv, top], numbers within the sequence, ascending, -1 behind the
    last.  q fp16 [R, Hq, 128]; row r is a query of sequence row_seq[r] (int32 [R]; None: r) that sees its first seq_lens[r]
    tokens (int32 [R]; a decode step's lengths with the new token, kv_step_plan's row_lens).  Where it sees more than `top`
    pages: the first `first` and the last `last` (1 at least) of them, and of the rest those whose bounds (kv_page_bounds) and
    k_scale allow the largest logit of any of the kv head's queries, in integers of 8 bits a value, ties to the lower page.
    Serves softmax scales above 0."""
    if bits != 8 and bits != 4:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    shape = bounds.shape
    if len(shape) != 4 or shape[2] != 2 or shape[3] != 16 * bits or bounds.element_size() != 1 or not bounds.is_contiguous():
        raise ValueError(f"bounds must be a contiguous 1-byte [P, Hkv, 2, {16 * bits}] tensor at {bits} bits, got "
                         f"{bounds.dtype} {tuple(shape)}")
    P, Hkv = shape[0], shape[1]
    if k_scale.dtype != torch.float16 or k_scale.shape != (P, Hkv) or not k_scale.is_contiguous():
        raise ValueError(f"k_scale must be a contiguous fp16 [{P}, {Hkv}] tensor")
    ld_q, R, Hq, B, max_pages = _check_rows(q, page_table, seq_lens, row_seq, Hkv)
    if last < 1 or first < 0 or first + last > top:
        raise ValueError(f"first = {first} and last = {last} (1 at least) of top = {top} pages")
    if out is not None:
        _check_out(out, (R, Hkv, top), q, (torch.int32,))
    index = _cuda_index(q, bounds, k_scale, page_table, seq_lens, row_seq)
    if not _current(index):
        with torch.cuda.device(index):
            return kv_select_pages(q, bounds, k_scale, page_table, seq_lens, bits, top, first, last, row_seq, out, workspace)
    if out is None:
        out = seq_lens.new_empty((R, Hkv, top))
    lib = _lib.load()
    ws = _call_workspace(workspace, lib.exl3_kv_select_workspace_bytes(R, Hkv, max_pages), q)
    _lib.check(lib.exl3_kv_select_pages(
        q.data_ptr(), ld_q, k_scale.data_ptr(), bounds.data_ptr(), P, page_table.data_ptr(), B, max_pages, _ptr(row_seq),
        seq_lens.data_ptr(), R, Hq, Hkv, _HEAD_DIM, 16, bits, top, first, last, out.data_ptr(), ws.data_ptr(), ws.nbytes,
        torch._C._cuda_getCurrentRawStream(index)), "kv_select_pages")
    return out


def kv_sparse_workspace_bytes(rows: int, num_q_heads: int, num_kv_heads: int, top: int) -> int:
    """Bytes of a `workspace` for kv_sparse_attention of up to `rows` rows (0: none of them need one)."""
    return _lib.load().exl3_kv_sparse_workspace_bytes(rows, num_q_heads, num_kv_heads, top)


def kv_sparse_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, bits: int,
                        pages: torch.Tensor, sm_scale: float | None = None, row_seq: torch.Tensor | None = None,
                        out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query row over the pages chosen for it.  q, page_table, seq_lens and row_seq as kv_select_pages has
    them, pages int32 [R, Hkv, top] as it returns them (or of another choice: distinct page numbers within the sequence; others
    are left out), the cache as kv_decode_attention has it.  A row that sees nothing gives zeros.  Returns fp16
    [R, Hq, 128]."""
    shape = k_cache.shape
    if bits != 8 and bits != 4:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    if len(shape) != 4 or shape != v_cache.shape or shape[2] != 16 or shape[3] != 16 * bits:
        raise ValueError(f"k_cache / v_cache must both be [P, Hkv, 16, {16 * bits}] at {bits} bits, got "
                         f"{tuple(shape)} / {tuple(v_cache.shape)}")
    if k_cache.element_size() != 1 or v_cache.element_size() != 1:
        raise ValueError("caches must hold 1-byte codes (int8 / uint8)")
    P, Hkv = shape[0], shape[1]
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != torch.float16 or t.shape != (P, Hkv) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp16 [{P}, {Hkv}] tensor")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    ld_q, R, Hq, B, max_pages = _check_rows(q, page_table, seq_lens, row_seq, Hkv)
    p_shape = pages.shape
    if pages.dtype != torch.int32 or len(p_shape) != 3 or p_shape[:2] != (R, Hkv) or not pages.is_contiguous():
        raise ValueError(f"pages must be a contiguous int32 [{R}, {Hkv}, top] tensor, got {pages.dtype} {tuple(p_shape)}")
    top = p_shape[2]
    if out is not None:
        _check_out(out, (R, Hq, _HEAD_DIM), q, _FP16)
    index = _cuda_index(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, pages, row_seq)
    if sm_scale is None:
        sm_scale = _HEAD_DIM ** -0.5
    if not _current(index):
        with torch.cuda.device(index):
            return kv_sparse_attention(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, bits, pages, sm_scale,
                                       row_seq, out, workspace)
    if out is None:
        out = q.new_empty((R, Hq, _HEAD_DIM))
    lib = _lib.load()
    need = lib.exl3_kv_sparse_workspace_bytes(R, Hq, Hkv, top)
    at = size = 0
    if need:
        ws = _call_workspace(workspace, need, q)
        at, size = ws.data_ptr(), ws.nbytes
    _lib.check(lib.exl3_kv_sparse_attention(
        q.data_ptr(), ld_q, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P,
        page_table.data_ptr(), B, max_pages, _ptr(row_seq), seq_lens.data_ptr(), R, Hq, Hkv, _HEAD_DIM, 16, bits,
        pages.data_ptr(), top, sm_scale, out.data_ptr(), at, size, torch._C._cuda_getCurrentRawStream(index)),
        "kv_sparse_attention")
    return out


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    """Bytes of a `workspace` for sample_tokens and sampling_probs of up to `rows` rows (no more for more than 512)."""
    return _lib.load().exl3_sample_workspace_bytes(rows, vocab)


def _setting(value, name: str, dtype: torch.dtype, lead: tuple, tensors: list) -> tuple[int | None, float]:
    """A setting of every row (a number), or one a row (a tensor): (pointer, number)."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.dtype != dtype or value.shape != lead or not value.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of shape {tuple(lead)}, got {value.dtype} "
                         f"{tuple(value.shape)}")
    tensors.append(value)
    return value.data_ptr(), 0


def _sample(what: str, logits: torch.Tensor, uniform: torch.Tensor | None, temperature, top_k, top_p, min_p, want_probs: bool,
            probs: torch.Tensor | None, workspace: torch.Tensor | None):
    shape = logits.shape
    if logits.dtype not in _WEIGHT_TYPE or len(shape) < 1:
        raise ValueError(f"logits must be fp16, bf16 or fp32 [..., V], got {logits.dtype} {tuple(shape)}")
    lead, V = shape[:-1], shape[-1]
    if len(shape) == 2:
        rows, ld = shape[0], logits.stride(0)
        if logits.stride(1) != 1 and V > 1:
            raise ValueError(f"logits: a row must be contiguous, got strides {logits.stride()}")
        ld = ld if rows > 1 else V
    else:
        if not logits.is_contiguous():
            raise ValueError("logits of other than two dimensions must be contiguous")
        rows, ld = logits.numel() // max(V, 1), V
    tensors = [logits]
    at_u = None
    if uniform is not None:
        if uniform.dtype != torch.float32 or uniform.shape != lead or not uniform.is_contiguous():
            raise ValueError(f"uniform must be a contiguous fp32 tensor of shape {tuple(lead)}")
        tensors.append(uniform)
        at_u = uniform.data_ptr()
    at_t, all_t = _setting(temperature, "temperature", torch.float32, lead, tensors)
    at_k, all_k = _setting(top_k, "top_k", torch.int32, lead, tensors)
    at_p, all_p = _setting(top_p, "top_p", torch.float32, lead, tensors)
    at_m, all_m = _setting(min_p, "min_p", torch.float32, lead, tensors)
    if not all_t >= 0 or not 0 <= all_p or not 0 <= all_m <= 1 or all_k < 0:
        raise ValueError(f"temperature = {all_t}, top_k = {all_k}, top_p = {all_p}, min_p = {all_m}")
    if probs is not None:
        _check_out(probs, shape, logits, (torch.float32,))
    index = _cuda_index(*tensors)
    if not _current(index):
        with torch.cuda.device(index):
            return _sample(what, logits, uniform, temperature, top_k, top_p, min_p, want_probs, probs, workspace)
    tokens = None if uniform is None else logits.new_empty(lead, dtype=torch.int32)
    if probs is None and want_probs:
        probs = logits.new_empty(shape, dtype=torch.float32)
    lib = _lib.load()
    need = lib.exl3_sample_workspace_bytes(rows, V)
    ws = _call_workspace(workspace, need, logits)
    _lib.check(lib.exl3_sample(
        logits.data_ptr(), _WEIGHT_TYPE[logits.dtype], ld, rows, V, at_u, at_t, all_t, at_k, min(all_k, V), at_p, all_p, at_m,
        all_m, _ptr(tokens), _ptr(probs), ws.data_ptr(), ws.nbytes, torch._C._cuda_getCurrentRawStream(index)), what)
    return tokens, probs


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  return_probs: bool = False, probs: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """Tokens drawn from logits fp16|bf16|fp32 [..., V] by given random numbers: with w = exp((l - max l) / temperature) and a
    row's elements in order of falling logits (ties by rising index), kept is the shortest of the first top_k (0: all), those
    whose predecessors have less than top_p of the first top_k's sum of w, and those with w >= min_p; the first element always.
    The token is the smallest one whose running sum of w over the kept passes uniform (fp32 [...], in [0, 1)) times their sum.
    Each setting is a number or a tensor [...] (fp32; top_k int32) with a value a row; temperature 0 takes the largest logit, the
    lowest of equals; NaN logits count as -inf; a row without a logit above -inf gives -1.
    Returns int32 [...], and with return_probs (or `probs` to write to) the distribution drawn from, fp32 [..., V]: what
    verify_drafts takes as draft_probs."""
    tokens, probs = _sample("sample_tokens", logits, uniform, temperature, top_k, top_p, min_p,
                            return_probs, probs, workspace)
    return tokens if probs is None else (tokens, probs)


def sampling_probs(logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The distribution that sample_tokens draws from with these settings, fp32 [..., V]: what verify_drafts takes as
    target_probs (a row without a logit above -inf: zeros)."""
    return _sample("sampling_probs", logits, None, temperature, top_k, top_p, min_p, True, out, workspace)[1]
