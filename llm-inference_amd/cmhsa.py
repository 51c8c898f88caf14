"""ctypes view of the C ABI in include/*.h (libcmhsa_hip.so).

This is the host-side plumbing only: device memory and streams come from PyTorch-ROCm, the
arithmetic is entirely in the hand-written gfx950 kernels.  There is NO fallback: if the library
is missing or no GPU is present, the calls raise.

  attention_fwd / attention_fwd_raw      cmhsa_fp32_fwd            full-sequence causal attention (the hot path)
  attention_fwd(..., workspace=ws)       cmhsa_fp32_fwd_ws         the same with a device workspace (class Workspace): query
                                                                   blocks may then be split across workgroups
  attention_fwd_packed_qkv               cmhsa_fp32_fwd_packed_qkv the same over one packed (.., T, 3*d_model) buffer
  decode_step                            cmhsa_fp32_decode_step    one-token step over a KV cache (opt-in)
  attention_packed_fwd                   cmhsa_packed_fwd          packed sequences, grouped heads, fp32 / bf16 / fp16
  kv4_append, kv4_gather, kv4_decode,    cmhsa_kv4_*               the paged 4-bit cache: store, read back, single-token
  kv4_copy_pages                                                   attention, page copies
  gelu_tanh_fwd                          gpt2_gelu_tanh_f32_fwd    fused tanh-GELU
  sustained_shader_clock_mhz             cmhsa_probe_shader_clock  measurement aid

The torch ops of the sibling extension module `causal_multihead_self_attention` (importing it registers them,
as the reference does at causal_self_attention.py:60-63) go through the same entry points; tests call both.
"""
from __future__ import annotations

import ctypes
import os

import torch  # must be imported BEFORE the library: both must share torch's libamdhip64

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libcmhsa_hip.so")

# every symbol include/*.h declares; tests/test_abi.py checks the headers against this list
EXPORTED_SYMBOLS = (
    "cmhsa_status_string",
    "cmhsa_version",
    "cmhsa_fp32_fwd",
    "cmhsa_fp32_fwd_ws",
    "cmhsa_fp32_fwd_noalloc",
    "cmhsa_workspace_bytes",
    "cmhsa_workspace_init",
    "cmhsa_fp32_fwd_workspace_bytes",
    "cmhsa_plan_describe",
    "cmhsa_plan_dump",
    "cmhsa_fp32_fwd_2d",
    "cmhsa_fp32_fwd_packed_qkv",
    "cmhsa_fp32_decode_step",
    "cmhsa_decode_algorithmic_bytes",
    "cmhsa_algorithmic_flops",
    "cmhsa_probe_shader_clock",
    "cmhsa_packed_workspace_bytes",  # include/cmhsa_packed.h
    "cmhsa_packed_fwd",
    "cmhsa_kv4_append",              # include/cmhsa_kv4.h
    "cmhsa_kv4_gather",
    "cmhsa_kv4_decode_workspace_bytes",
    "cmhsa_kv4_decode",
    "cmhsa_kv4_copy_pages",
    "gpt2_gelu_tanh_f32_fwd",        # include/gpt2_gelu.h
    "gpt2_gelu_algorithmic_bytes",
    "gpt2_add_layernorm_f32_fwd",    # include/gpt2_layernorm.h
    "gpt2_add_layernorm_algorithmic_bytes",
    "gpt2_embed_f32_fwd",            # include/gpt2_step.h
    "gpt2_greedy_step",
    "gpt2_linear_rows_f32_fwd",      # include/gpt2_linear.h
    "gpt2_ln_linear_rows_f32_fwd",
    "gpt2_linear_rows_algorithmic_bytes",
)

CMHSA_OK = 0
CMHSA_ERR_NULL_POINTER = -1
CMHSA_ERR_BAD_SHAPE = -2
CMHSA_ERR_HEAD_DIM = -3
CMHSA_ERR_ALIGNMENT = -4
CMHSA_ERR_TOO_LARGE = -5
CMHSA_ERR_WORKSPACE = -6
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # CMHSA_F32 / CMHSA_BF16 / CMHSA_F16 (include/cmhsa_packed.h)
NOALLOC_SCRATCH_BYTES = 1 << 20          # CMHSA_NOALLOC_SCRATCH_BYTES (include/cmhsa.h)

_lib = None


class CmhsaError(RuntimeError):
    def __init__(self, status: int, text: str):
        super().__init__(f"cmhsa status {status}: {text}")
        self.status = status


def load_library() -> ctypes.CDLL:
    """dlopen libcmhsa_hip.so (once) and declare the prototypes of include/cmhsa.h."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise FileNotFoundError(
            f"{LIB_PATH} is missing: build it with `python llm-inference_amd/build.py` "
            "(there is no CPU or PyTorch fallback for the HIP attention path)")
    lib = ctypes.CDLL(LIB_PATH)
    i64, i32, vp, sz = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t
    lib.cmhsa_status_string.restype = ctypes.c_char_p
    lib.cmhsa_status_string.argtypes = [i32]
    lib.cmhsa_version.restype = i32
    lib.cmhsa_version.argtypes = []
    lib.cmhsa_fp32_fwd.restype = i32
    lib.cmhsa_fp32_fwd.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, i64, i32, i32, i32, i32, vp]
    lib.cmhsa_fp32_fwd_ws.restype = i32
    lib.cmhsa_fp32_fwd_ws.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, i64, i32, i32, i32, i32, vp, sz, vp]
    lib.cmhsa_fp32_fwd_noalloc.restype = i32
    lib.cmhsa_fp32_fwd_noalloc.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, i64, i32, i32, i32, i32, vp]
    lib.cmhsa_workspace_bytes.restype = sz
    lib.cmhsa_workspace_bytes.argtypes = []
    lib.cmhsa_workspace_init.restype = i32
    lib.cmhsa_workspace_init.argtypes = [vp, sz, vp]
    lib.cmhsa_fp32_fwd_workspace_bytes.restype = sz
    lib.cmhsa_fp32_fwd_workspace_bytes.argtypes = [i32, i32, i32]
    lib.cmhsa_plan_describe.restype = i32
    lib.cmhsa_plan_describe.argtypes = [i32, i32, i32, i32, ctypes.c_char_p, i32]
    lib.cmhsa_plan_dump.restype = i32
    lib.cmhsa_plan_dump.argtypes = [i32, i32, i32, i32, i32, ctypes.POINTER(ctypes.c_int), i32]
    lib.cmhsa_fp32_fwd_2d.restype = i32
    lib.cmhsa_fp32_fwd_2d.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i32, i32, i32, vp]
    lib.cmhsa_fp32_fwd_packed_qkv.restype = i32
    lib.cmhsa_fp32_fwd_packed_qkv.argtypes = [vp, vp, i64, i64, i64, i64, i32, i32, i32, i32, vp, sz, vp]
    lib.cmhsa_fp32_decode_step.restype = i32
    lib.cmhsa_fp32_decode_step.argtypes = [vp, i64, vp, vp, i64, i64, vp, i64, vp, i32, i32, i32, i32, vp]
    lib.cmhsa_decode_algorithmic_bytes.restype = ctypes.c_double
    lib.cmhsa_decode_algorithmic_bytes.argtypes = [i32, i32, i32, i32]
    lib.cmhsa_probe_shader_clock.restype = i32
    lib.cmhsa_probe_shader_clock.argtypes = [vp, i32, vp]
    lib.cmhsa_algorithmic_flops.restype = ctypes.c_double
    lib.cmhsa_algorithmic_flops.argtypes = [i32, i32, i32, i32]
    lib.gpt2_gelu_tanh_f32_fwd.restype = i32
    lib.gpt2_gelu_tanh_f32_fwd.argtypes = [vp, vp, i64, vp]
    lib.gpt2_gelu_algorithmic_bytes.restype = ctypes.c_double
    lib.gpt2_gelu_algorithmic_bytes.argtypes = [i64]
    lib.gpt2_add_layernorm_f32_fwd.restype = i32
    lib.gpt2_add_layernorm_f32_fwd.argtypes = [vp, vp, vp, vp, vp, vp, i64, i32, i64, i64, ctypes.c_float, vp]
    lib.gpt2_add_layernorm_algorithmic_bytes.restype = ctypes.c_double
    lib.gpt2_add_layernorm_algorithmic_bytes.argtypes = [i64, i32, i32]
    lib.gpt2_embed_f32_fwd.restype = i32
    lib.gpt2_embed_f32_fwd.argtypes = [vp, i64, vp, vp, vp, i32, i32, i32, i32, vp]
    lib.gpt2_greedy_step.restype = i32
    lib.gpt2_greedy_step.argtypes = [vp, i64, vp, vp, i64, vp, i32, i32, i32, i64, vp]
    lib.gpt2_linear_rows_f32_fwd.restype = i32
    lib.gpt2_linear_rows_f32_fwd.argtypes = [vp, i64, vp, i64, vp, vp, i64, i32, i32, i32, i32, vp]
    lib.gpt2_ln_linear_rows_f32_fwd.restype = i32
    lib.gpt2_ln_linear_rows_f32_fwd.argtypes = [vp, i64, vp, i64, vp, vp, ctypes.c_float, vp, vp, i64, vp, vp, i64, i32, i32, i32, i32, vp]
    lib.gpt2_linear_rows_algorithmic_bytes.restype = ctypes.c_double
    lib.gpt2_linear_rows_algorithmic_bytes.argtypes = [i32, i32, i32, i32]
    lib.cmhsa_packed_fwd.restype = i32
    lib.cmhsa_packed_fwd.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, vp, vp, i32, i32, i32, i32, i32, i32, i32, i32, vp, sz, vp]
    lib.cmhsa_packed_workspace_bytes.restype = sz
    lib.cmhsa_packed_workspace_bytes.argtypes = [i32, i32, i32, i32, i32, i32, i32]
    lib.cmhsa_kv4_append.restype = i32
    lib.cmhsa_kv4_append.argtypes = [vp, vp, i64, i64, i32, vp, i64, i32, i32, vp, i64, i32, vp, vp, i32, i32, i32, i32, vp]
    lib.cmhsa_kv4_gather.restype = i32
    lib.cmhsa_kv4_gather.argtypes = [vp, vp, i64, i64, i32, vp, i64, i32, i32, vp, i64, i32, vp, vp, i32, i32, i32, i32, i32, vp]
    lib.cmhsa_kv4_decode_workspace_bytes.restype = sz
    lib.cmhsa_kv4_decode_workspace_bytes.argtypes = [i32, i32, i32, i32, i32, i32]
    lib.cmhsa_kv4_decode.restype = i32
    lib.cmhsa_kv4_decode.argtypes = [vp, vp, i64, i64, i32, vp, i64, i32, i32, vp, i64, i32, vp, i32, i32, i32, i32, vp, sz, vp]
    lib.cmhsa_kv4_copy_pages.restype = i32
    lib.cmhsa_kv4_copy_pages.argtypes = [vp, i64, i32, i64, i32, i64, ctypes.POINTER(i32), ctypes.POINTER(i32), i32, vp]
    _lib = lib
    return lib


def status_string(status: int) -> str:
    return load_library().cmhsa_status_string(status).decode()


def algorithmic_flops(batch: int, seq_len: int, num_heads: int, head_dim: int = 64) -> float:
    """F = 2*B*H*d*T*(T+1); pure host arithmetic, no GPU needed."""
    return float(load_library().cmhsa_algorithmic_flops(batch, seq_len, num_heads, head_dim))


def plan_dump(batch: int, seq_len: int, num_heads: int, with_workspace: bool = False, cus: int = 0) -> dict:
    """The plan of a shape as data (cmhsa_plan_dump; no GPU needed when `cus` is given): header fields and, per workgroup
    of a (b,h), its segments as (n, first_unit, unit_count, wave_mask, part_word) tuples (absent segments dropped)."""
    lib = load_library()
    need = lib.cmhsa_plan_dump(batch, seq_len, num_heads, 1 if with_workspace else 0, cus, None, 0)
    if need <= 0:
        raise CmhsaError(need, status_string(need))
    buf = (ctypes.c_int * need)()
    got = lib.cmhsa_plan_dump(batch, seq_len, num_heads, 1 if with_workspace else 0, cus, buf, need)
    if got != need:
        raise CmhsaError(got, status_string(got))
    names = ("waves", "segs", "wgs_per_bh", "grid_x", "grid_y", "grid_z", "parts_per_bh", "splits_per_bh", "simd_cap", "nqb",
             "use_table", "longest_first", "chain", "n_paired", "n_alone", "workspace_256")
    plan = dict(zip(names, buf[:16]))
    if plan["use_table"] == 2:
        # the 16-row-block family (csrc/cmhsa_tiles16.h): "segs" = job words per wave, "nqb" = 16-row blocks per (b,h),
        # "simd_cap" = tiles on the busiest SIMD; per workgroup its 4 or 8 job lists in run order (with 8 waves the lists
        # 2s and 2s + 1 share SIMD s), per list its jobs as (block, first_tile, tiles, rank, pieces); "merges" = per
        # workgroup, the barrier flag of each list's first word
        J, W = plan["segs"], plan["waves"]
        plan.update(family="tiles16", jobs_per_wave=J, blocks=plan["nqb"], tiles_per_simd=plan["simd_cap"], sub=plan["chain"],
                    contig=bool(plan["n_paired"]))
        words = [[[buf[16 + (j * W + w) * J + i] & 0xffffffff for i in range(J)] for w in range(W)] for j in range(plan["wgs_per_bh"])]
        gran = max(1, plan["n_alone"])                     # tiles per count of a job word's first-tile / tiles fields
        plan["granule"] = gran
        plan["workgroups"] = [[[(x & 255, gran * ((x >> 8) & 255), gran * ((x >> 16) & 255), (x >> 24) & 7, (x >> 27) & 15) for x in wave if (x >> 16) & 255]
                               for wave in wg] for wg in words]
        plan["merges"] = [[bool(wave[0] >> 31) for wave in wg] for wg in words]
        plan["raw_words"] = words
        return plan
    if plan["use_table"] == 3:
        # job lists (one-wave workgroups, the kernel's kList variant): "chain" = (b,h)s per period, "n_paired" = lists per
        # period (= grid_y), "simd_cap" = units of the longest list; per list its jobs as (units of the block = block index
        # + 1, (b,h) within the period); "descending_up_to" = blocks of at most that many units are taken from the diagonal
        # unit down.  Period P = 8 * z + x of the grid covers the (b,h)s [P * period_bh, (P + 1) *
        # period_bh) that exist; a list's entries whose (b,h) does not exist are dropped by the kernel.
        plan.update(family="lists", period_bh=plan["chain"], lists_per_period=plan["n_paired"], units_per_list=plan["simd_cap"],
                    jobs_per_list=plan["n_alone"], descending_up_to=plan["workspace_256"], workspace_256=0)
        words = [[buf[16 + l * 8 + i] & 0xffffffff for i in range(8)] for l in range(plan["lists_per_period"])]
        entries = [[(w >> (16 * h)) & 0xffff for w in ws for h in (0, 1)] for ws in words]
        plan["lists"] = [[(e & 255, e >> 8) for e in es if e & 255] for es in entries]
        plan["raw_words"] = words
        return plan
    plan["family"] = "units32"
    segs = plan["segs"]
    plan["workgroups"] = [[tuple(buf[16 + (j * segs + i) * 5: 16 + (j * segs + i) * 5 + 5]) for i in range(segs)
                           if buf[16 + (j * segs + i) * 5] != 0] for j in range(plan["wgs_per_bh"])]
    return plan


def plan_description(batch: int, seq_len: int, num_heads: int, workspace_bytes: int = 0) -> str:
    """One line on the plan the library uses for this shape on the current device (cmhsa_plan_describe)."""
    buf = ctypes.create_string_buffer(512)
    rc = load_library().cmhsa_plan_describe(batch, seq_len, num_heads, 1 if workspace_bytes > 0 else 0, buf, len(buf))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return buf.value.decode()


class Workspace:
    """Device workspace of cmhsa_fp32_fwd_ws: CMHSA_WORKSPACE_BYTES of torch-allocated (hipMalloc'd) device memory whose
    counter block is zeroed once, on torch's current stream.  One per stream: calls that overlap in time on one GPU must
    not share it."""

    def __init__(self, device=None):
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        lib = load_library()
        self.nbytes = int(lib.cmhsa_workspace_bytes())
        self.buffer = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        if self.buffer.data_ptr() % 256:
            raise RuntimeError("allocator returned memory that is not 256-byte aligned")
        self.ptr = ctypes.c_void_p(self.buffer.data_ptr())
        self.device = device
        self.reset()

    def reset(self) -> None:
        """Zero the counter block again (only needed after a launch that did not run to completion)."""
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream(self.device).cuda_stream
            rc = load_library().cmhsa_workspace_init(self.ptr, self.nbytes, ctypes.c_void_p(stream))
        if rc != CMHSA_OK:
            raise CmhsaError(rc, status_string(rc))


def _check(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32")
    if t.dim() not in (2, 3):
        raise ValueError(f"{name} must be a 2D (N, d_model) or 3D (B, N, d_model) tensor")
    if t.stride(-1) != 1:
        raise ValueError(f"{name}'s last-dim stride must be 1")


def attention_fwd_raw(q_ptr: int, k_ptr: int, v_ptr: int, o_ptr: int,
                      row_strides, batch_strides, batch: int, seq_len: int, num_heads: int, head_dim: int,
                      stream: int = 0) -> int:
    """Direct call of cmhsa_fp32_fwd with raw device addresses; returns the status code."""
    return load_library().cmhsa_fp32_fwd(
        q_ptr, k_ptr, v_ptr, o_ptr, *[int(s) for s in row_strides], *[int(s) for s in batch_strides],
        batch, seq_len, num_heads, head_dim, ctypes.c_void_p(stream))


def attention_fwd(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, num_heads: int,
                  out: torch.Tensor | None = None, workspace: "Workspace | None" = None) -> torch.Tensor:
    """Causal multi-head self-attention forward through the C ABI, on torch's current stream.

    Q, K, V: (N, d_model) or (B, N, d_model) fp32 device tensors, last-dim stride 1, arbitrary
    row stride (multiple of 4).  Returns a new contiguous tensor unless `out` is given.
    With `workspace` the call goes through cmhsa_fp32_fwd_ws (query blocks may be split across workgroups).
    """
    for t, n in ((Q, "Q"), (K, "K"), (V, "V")):
        _check(t, n)
    if K.shape != Q.shape or V.shape != Q.shape:
        raise ValueError("Q, K and V must have the same shape")
    d_model = Q.shape[-1]
    if num_heads <= 0 or d_model % num_heads != 0:
        raise ValueError("Feature dimension of Q must be evenly divisible by the number of heads")
    if out is None:
        out = torch.empty(Q.shape, dtype=torch.float32, device=Q.device)
    batched = Q.dim() == 3
    B = Q.shape[0] if batched else 1
    N = Q.shape[-2]
    bs = [t.stride(0) if batched else 0 for t in (Q, K, V, out)]
    rs = [t.stride(-2) for t in (Q, K, V, out)]
    with torch.cuda.device(Q.device):
        stream = torch.cuda.current_stream(Q.device).cuda_stream
        if workspace is not None:
            if workspace.device != Q.device:
                raise ValueError("workspace is on another device")
            rc = load_library().cmhsa_fp32_fwd_ws(
                Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), *[int(x) for x in rs], *[int(x) for x in bs],
                B, N, num_heads, d_model // num_heads, workspace.ptr, workspace.nbytes, ctypes.c_void_p(stream))
        else:
            rc = attention_fwd_raw(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), rs, bs,
                                   B, N, num_heads, d_model // num_heads, stream)
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def attention_fwd_packed_qkv(QKV: torch.Tensor, num_heads: int, workspace: "Workspace | None" = None) -> torch.Tensor:
    """cmhsa_fp32_fwd_packed_qkv: QKV is the (N, 3*d_model) or (B, N, 3*d_model) output of the fused QKV linear layer
    (row = [Q | K | V], reference causal_self_attention.py:224-227); returns the (.., N, d_model) context."""
    _check(QKV, "QKV")
    if num_heads <= 0 or QKV.shape[-1] % (3 * num_heads) != 0:
        raise ValueError("last dimension of QKV must be 3 * d_model with d_model divisible by the number of heads")
    d_model = QKV.shape[-1] // 3
    out = torch.empty(QKV.shape[:-1] + (d_model,), dtype=torch.float32, device=QKV.device)
    batched = QKV.dim() == 3
    with torch.cuda.device(QKV.device):
        stream = torch.cuda.current_stream(QKV.device).cuda_stream
        rc = load_library().cmhsa_fp32_fwd_packed_qkv(
            QKV.data_ptr(), out.data_ptr(), QKV.stride(-2), out.stride(-2),
            QKV.stride(0) if batched else 0, out.stride(0) if batched else 0,
            QKV.shape[0] if batched else 1, QKV.shape[-2], num_heads, d_model // num_heads,
            workspace.ptr if workspace is not None else None, workspace.nbytes if workspace is not None else 0, ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def decode_step(qkv_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, num_heads: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """cmhsa_fp32_decode_step (opt-in KV-cache mode): qkv_new (B, 3*d_model) of the new token, caches (B, capacity,
    d_model) updated in place at row `pos` (int32 device tensor, one element); returns the (B, d_model) context."""
    for t in (qkv_new, k_cache, v_cache):
        if not t.is_cuda or t.dtype != torch.float32 or t.stride(-1) != 1:
            raise ValueError("qkv_new, k_cache and v_cache must be float32 CUDA tensors with last-dim stride 1")
    if not pos.is_cuda or pos.dtype != torch.int32 or pos.numel() != 1:
        raise ValueError("pos must be an int32 CUDA tensor with one element")
    if qkv_new.dim() != 2 or k_cache.dim() != 3 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("qkv_new must be (B, 3*d_model); k_cache and v_cache (B, capacity, d_model) with equal strides")
    B, d_model = qkv_new.shape[0], qkv_new.shape[1] // 3
    if num_heads <= 0 or qkv_new.shape[1] != 3 * d_model or d_model % num_heads or k_cache.shape[0] != B or k_cache.shape[2] != d_model:
        raise ValueError("shape mismatch between qkv_new, the caches and num_heads")
    if out is None:
        out = torch.empty((B, d_model), dtype=torch.float32, device=qkv_new.device)
    with torch.cuda.device(qkv_new.device):
        stream = torch.cuda.current_stream(qkv_new.device).cuda_stream
        rc = load_library().cmhsa_fp32_decode_step(
            qkv_new.data_ptr(), qkv_new.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(1), k_cache.stride(0),
            out.data_ptr(), out.stride(0), pos.data_ptr(), B, k_cache.shape[1], num_heads, d_model // num_heads,
            ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def sustained_shader_clock_mhz(device=None, iters: int = 2000) -> float:
    """Shader clock (MHz) the chip sustains while every CU runs fp32 MFMA chains: cmhsa_probe_shader_clock."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    out = torch.zeros(4, dtype=torch.int64, device=device)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        for _ in range(2):                                   # the first pass ramps the clocks, the second is read
            rc = load_library().cmhsa_probe_shader_clock(out.data_ptr(), iters, ctypes.c_void_p(stream))
            if rc != CMHSA_OK:
                raise CmhsaError(rc, status_string(rc))
        torch.cuda.synchronize(device)
    t0, t1, r0, r1 = (int(x) for x in out.tolist())
    return (t1 - t0) / max(r1 - r0, 1) * 100.0


def gelu_tanh_fwd(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused tanh-GELU (reference gelu.py:8-12) through the C ABI of include/gpt2_gelu.h, on torch's current
    stream.  x: contiguous fp32 device tensor of any shape; `out` may be x itself (in place)."""
    if not x.is_cuda or x.dtype != torch.float32:
        raise ValueError("x must be a float32 CUDA tensor")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError("out must match x (shape, dtype, device) and be contiguous")
    with torch.cuda.device(x.device):
        stream = torch.cuda.current_stream(x.device).cuda_stream
        rc = load_library().gpt2_gelu_tanh_f32_fwd(x.data_ptr(), out.data_ptr(), x.numel(), ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def _check_packed(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in DTYPE_CODES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be 2D (rows, heads * head_dim) with last-dim stride 1")
    if like is not None and (t.device != like.device or t.dtype != like.dtype):
        raise ValueError(f"{name} must be on the same device and of the same type as the other tensors")


def _stride(t: torch.Tensor, dim: int, dense: int) -> int:
    """t's stride over `dim`; `dense` where there is one row (page, layer) at most and its stride means nothing."""
    return t.stride(dim) if t.shape[dim] > 1 else dense


def _row_stride(t: torch.Tensor) -> int:
    return _stride(t, 0, -(-t.shape[1] // 8) * 8)


def _check_ints(t: torch.Tensor, name: str, like: torch.Tensor, count: int | None = None) -> None:
    if t.device != like.device or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1D int32 tensor on the same device")
    if count is not None and t.numel() != count:
        raise ValueError(f"{name} must have {count} elements")


def attention_packed_fwd(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor, num_heads: int,
                         num_kv_heads: int, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """cmhsa_packed_fwd: Q (rows, num_heads * D), K / V (rows, num_kv_heads * D), sequence s = rows cu_q[s] .. cu_q[s+1]-1 of Q and
    cu_k[s] .. cu_k[s+1]-1 of K / V; the last query row of a sequence sees its last key.  Rows behind the last sequence are
    left as they were in a given `out`, and zero in one that this call makes.  `workspace`: a uint8 tensor of
    cmhsa_packed_workspace_bytes, for shapes whose keys may be cut between workgroups; without one they are not cut."""
    _check_packed(Q, "Q")
    _check_packed(K, "K", Q)
    _check_packed(V, "V", Q)
    if num_heads <= 0 or num_kv_heads <= 0 or Q.shape[1] % num_heads:
        raise ValueError("Feature dimension of Q must be evenly divisible by the number of heads")
    d = Q.shape[1] // num_heads
    if K.shape != V.shape or K.shape[1] != num_kv_heads * d:
        raise ValueError("K and V must both be (rows, num_kv_heads * head_dim)")
    _check_ints(cu_q, "cu_q", Q)
    _check_ints(cu_k, "cu_k", Q, cu_q.numel())
    if cu_q.numel() < 1:
        raise ValueError("cu_q must have an element more than there are sequences")
    given = out is not None
    if given:
        _check_packed(out, "out", Q)
        if out.shape != Q.shape:
            raise ValueError("out must have Q's shape")
    else:
        out = torch.empty(Q.shape, dtype=Q.dtype, device=Q.device)
    if workspace is not None and (workspace.device != Q.device or workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous uint8 tensor on the same device")
    with torch.cuda.device(Q.device):
        stream = torch.cuda.current_stream(Q.device).cuda_stream
        rc = load_library().cmhsa_packed_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), _row_stride(Q), _row_stride(K), _row_stride(V), _row_stride(out),
                                             cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, Q.shape[0], K.shape[0], num_heads, num_kv_heads, d,
                                             DTYPE_CODES[Q.dtype], 0 if given else 1, None if workspace is None else workspace.data_ptr(),
                                             0 if workspace is None else workspace.numel(), ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def kv4_block_bytes(page_size: int, head_dim: int) -> int:
    """CMHSA_KV4_BLOCK_BYTES: bytes that one page holds of one K/V head."""
    return page_size * head_dim // 16 * 17


def _check_pages(pages: torch.Tensor, head_dim: int, page_table: torch.Tensor, num_seqs: int, like: torch.Tensor) -> int:
    """The page size of a pool (num_pages, num_kv_heads, block bytes) on like's device, checked against the table of `num_seqs` sequences."""
    if pages.device != like.device:
        raise ValueError("pages must be on the same device as the other tensors")
    if not pages.is_cuda or pages.dtype != torch.uint8 or pages.dim() != 3 or pages.stride(2) != 1 or (pages.shape[1] > 1 and pages.stride(1) != pages.shape[2]):
        raise ValueError("pages must be a (num_pages, num_kv_heads, block bytes) uint8 CUDA tensor with contiguous pages")
    page_size = pages.shape[2] * 16 // (17 * head_dim) if head_dim > 0 else 0
    if page_size <= 0 or kv4_block_bytes(page_size, head_dim) != pages.shape[2]:
        raise ValueError("pages' last dimension must be page_size * head_dim * 17 / 16 bytes")
    if page_table.device != pages.device or page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != num_seqs or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be a (sequences, pages) int32 tensor with contiguous rows on the same device")
    return page_size


def kv4_append(K: torch.Tensor, V: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
               starts: torch.Tensor | None = None) -> None:
    """cmhsa_kv4_append: row r of K / V (rows, num_kv_heads * D), of sequence s, to position starts[s] + r - cu_seqlens[s] of its pages."""
    _check_packed(K, "K")
    _check_packed(V, "V", K)
    if pages.dim() != 3 or pages.shape[1] < 1 or K.shape != V.shape or K.shape[1] % pages.shape[1]:
        raise ValueError("K and V must both be (rows, pages.shape[1] * head_dim)")
    _check_ints(cu_seqlens, "cu_seqlens", K)
    n, d = cu_seqlens.numel() - 1, K.shape[1] // pages.shape[1]
    page_size = _check_pages(pages, d, page_table, n, K)
    if starts is not None:
        _check_ints(starts, "starts", K, n)
    with torch.cuda.device(K.device):
        stream = torch.cuda.current_stream(K.device).cuda_stream
        rc = load_library().cmhsa_kv4_append(K.data_ptr(), V.data_ptr(), _row_stride(K), _row_stride(V), DTYPE_CODES[K.dtype], pages.data_ptr(), _stride(pages, 0, pages.shape[1] * pages.shape[2]), pages.shape[0],
                                             page_size, page_table.data_ptr(), page_table.stride(0), page_table.shape[1], cu_seqlens.data_ptr(),
                                             None if starts is None else starts.data_ptr(), n, K.shape[0], pages.shape[1], d, ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))


def kv4_gather(pages: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor, starts: torch.Tensor | None, head_dim: int,
               out: tuple[torch.Tensor, torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    """cmhsa_kv4_gather into the given (K, V), each (rows, num_kv_heads * head_dim); rows behind the last sequence are left as they were."""
    K, V = out
    _check_packed(K, "K")
    _check_packed(V, "V", K)
    if pages.dim() != 3 or K.shape != V.shape or K.shape[1] != pages.shape[1] * head_dim:
        raise ValueError("K and V must both be (rows, pages.shape[1] * head_dim)")
    _check_ints(cu_seqlens, "cu_seqlens", K)
    n = cu_seqlens.numel() - 1
    page_size = _check_pages(pages, head_dim, page_table, n, K)
    if starts is not None:
        _check_ints(starts, "starts", K, n)
    with torch.cuda.device(K.device):
        stream = torch.cuda.current_stream(K.device).cuda_stream
        rc = load_library().cmhsa_kv4_gather(K.data_ptr(), V.data_ptr(), _row_stride(K), _row_stride(V), DTYPE_CODES[K.dtype], pages.data_ptr(), _stride(pages, 0, pages.shape[1] * pages.shape[2]), pages.shape[0],
                                             page_size, page_table.data_ptr(), page_table.stride(0), page_table.shape[1], cu_seqlens.data_ptr(),
                                             None if starts is None else starts.data_ptr(), n, K.shape[0], pages.shape[1], head_dim, 0, ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def kv4_decode(q: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, num_heads: int,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """cmhsa_kv4_decode: q (sequences, num_heads * D), one token a sequence over the first lengths[s] positions of its pages.
    `workspace`: a uint8 tensor to use instead of one that this call allocates."""
    _check_packed(q, "q")
    if num_heads <= 0 or q.shape[1] % num_heads or pages.dim() != 3 or pages.shape[1] < 1:
        raise ValueError("Feature dimension of q must be evenly divisible by the number of heads")
    n, d = q.shape[0], q.shape[1] // num_heads
    page_size = _check_pages(pages, d, page_table, n, q)
    _check_ints(lengths, "lengths", q, n)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_packed(out, "out", q)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
    lib = load_library()
    if workspace is None:
        workspace = torch.empty(lib.cmhsa_kv4_decode_workspace_bytes(n, page_table.shape[1], page_size, num_heads, pages.shape[1], d), dtype=torch.uint8, device=q.device)
    elif workspace.device != q.device or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the same device")
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream(q.device).cuda_stream
        rc = lib.cmhsa_kv4_decode(q.data_ptr(), out.data_ptr(), _row_stride(q), _row_stride(out), DTYPE_CODES[q.dtype], pages.data_ptr(), _stride(pages, 0, pages.shape[1] * pages.shape[2]), pages.shape[0],
                                  page_size, page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(), n, num_heads, pages.shape[1], d,
                                  workspace.data_ptr(), workspace.numel(), ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
    return out


def kv4_copy_pages(pages: torch.Tensor, src, dst) -> None:
    """cmhsa_kv4_copy_pages: page dst[i] := page src[i] of (num_pages, num_kv_heads, block bytes) or (layers, num_pages, ..)."""
    if not pages.is_cuda or pages.dtype != torch.uint8 or pages.dim() not in (3, 4):
        raise ValueError("pages must be a uint8 CUDA tensor of 3 or 4 dimensions")
    if len(src) != len(dst):
        raise ValueError("src and dst must have the same number of pages")
    if pages.stride(-1) != 1 or (pages.shape[-2] > 1 and pages.stride(-2) != pages.shape[-1]):
        raise ValueError("a page's blocks must be contiguous")
    if not all(0 <= page < pages.shape[-3] for page in (*src, *dst)):      # (a ctypes int keeps the low 32 bits of what it is given)
        raise ValueError(f"src and dst must be page numbers below {pages.shape[-3]}")
    ints = ctypes.c_int * max(len(src), 1)
    with torch.cuda.device(pages.device):
        stream = torch.cuda.current_stream(pages.device).cuda_stream
        rc = load_library().cmhsa_kv4_copy_pages(pages.data_ptr(), _stride(pages, 0, 0) if pages.dim() == 4 else 0, pages.shape[0] if pages.dim() == 4 else 1,
                                                 _stride(pages, -3, pages.shape[-2] * pages.shape[-1]), pages.shape[-3], pages.shape[-2] * pages.shape[-1], ints(*src), ints(*dst), len(src), ctypes.c_void_p(stream))
    if rc != CMHSA_OK:
        raise CmhsaError(rc, status_string(rc))
