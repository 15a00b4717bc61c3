"""ctypes binding of libneuratensor_native.so (the C ABI in include/neuratensor_native.h).

Each wrapper takes torch CUDA tensors, checks them, allocates the outputs
and the workspace through torch's caching allocator and calls the C entry
point on the current CUDA stream.  There is no fallback: if the library is
missing or the tensors are not on an sm_100 GPU, the call raises.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import struct
import threading
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libneuratensor_native.so")

NT_F32, NT_BF16, NT_U8 = 0, 1, 2
_DT = {torch.float32: NT_F32, torch.bfloat16: NT_BF16}
_STATUS = {1: "bad argument", 2: "unsupported dtype", 3: "unsupported GPU", 4: "CUDA error",
           5: "device wait timed out", 6: "workspace too small"}


class NativeError(RuntimeError):
    """A libneuratensor_native call returned a non-zero status."""

    def __init__(self, fn: str, status: int, msg: str):
        super().__init__(f"{fn}: {msg or _STATUS.get(status, 'error')} (status {status})")
        self.status = status


_lib = None
_lock = threading.Lock()
_I64, _I32, _F32, _P = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_void_p

_SIGS = {
    "nt_abi_version": ([], _I32),
    "nt_last_error": ([], ctypes.c_char_p),
    "nt_device_supported": ([_I32], _I32),
    "nt_get_error_flag": ([_I32, ctypes.POINTER(ctypes.c_uint), _I32], _I32),
    "nt_launch_count": ([], ctypes.c_ulonglong),
    "nt_bounded_wait_check": ([_I64, _P], _I32),
    "nt_lif_scan": ([_I32, _I64, _I64, _I64, _P, _I64, _I64, _P, _P, _P, _P, _P, _I64, _I64, _P, _P], _I32),
    "nt_selective_scan": ([_I32, _I32, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P], _I32),
    "nt_ssm_workspace_bytes": ([_I32, _I64, _I64, _I64, _I64], _I64),
    "nt_ssm_forward": ([_I32, _I32, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _P], _I32),
    "nt_sparse_out_proj_workspace_bytes": ([_I32, _I64, _I64, _I64], _I64),
    "nt_sparse_out_proj": ([_I32, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _I64, _P], _I32),
    "nt_rmsnorm_in_proj_workspace_bytes": ([_I32, _I64, _I64, _I64], _I64),
    "nt_rmsnorm_in_proj": ([_I32, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _I64, _P], _I32),
    "nt_noalloc_scratch_bytes": ([], ctypes.c_size_t),
    "nt_rmsnorm_in_proj_noalloc": ([_I32, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P], _I32),
    "nt_block_workspace_bytes": ([_I32, _I64, _I64, _I64, _I64, _I64], _I64),
    "nt_block_forward": ([_I32, _I32, _I64, _I64, _I64, _I64, _I64] + [_P] * 17 + [_I32, _P, _I64, _P], _I32),
    "nt_lif_ssm_fused": ([_I64, _I64, _I64, _I64] + [_P] * 14 + [_I32, _P, _P], _I32),
    "nt_window_attention": ([_I32, _I64, _I64, _I64, _I64, _I64, _P, _I64, _P, _P, _P, _I64, _P], _I32),
    "nt_embedding": ([_I32, _I64, _I64, _I64, _P, _P, _P, _P], _I32),
    "nt_greedy_tokens": ([_I32, _I64, _I64, _P, _I64, _P, _P, _P], _I32),
    "nt_attention_workspace_bytes": ([_I32, _I64, _I64, _I64], _I64),
    "nt_attention_forward": ([_I32, _I64, _I64, _I64, _I64, _I64] + [_P] * 8 + [_I64, _P], _I32),
    "nt_attention_output": ([_I32, _I64, _I64] + [_P] * 5, _I32),
    "nt_lm_head_workspace_bytes": ([_I32, _I64, _I64, _I64], _I64),
    "nt_lm_head": ([_I32, _I64, _I64, _I64, _P, _P, _P, _P, _P, _I64, _P], _I32),
    "nt_rotary": ([_I32, _I64, _I64, _I64, _I64, _I64, _I32, _I32, _F32, _P, _I64, _I64, _I64, _P, _I64, _P, _P, _I64,
                   _I64, _I64, _P], _I32),
    "nt_kv_append": ([_I32] + [_I64] * 7 + [_P, _I64, _I64, _I64] * 2 + [_P] * 5 + [_I64, _P, _P, _P], _I32),
    "nt_kv_attention_workspace_bytes": ([_I64] * 8, _I64),
    "nt_kv_attention": ([_I32] + [_I64] * 9 + [_F32, _P, _I64, _I64, _I64] + [_P] * 5 + [_I64, _P, _P, _P, _P, _I64, _P],
                        _I32),
    "nt_logits_process": ([_I32, _I64, _I64, _P, _I64, _P, _I64, _I64, _P, _P, _I32, _P, ctypes.c_double] + [_P, _F32] * 2 +
                          [_P, _I64, _P, _I64, _I64, _P, _I64, _P, _I64, _P], _I32),
    "nt_beam_select_workspace_bytes": ([_I32] + [_I64] * 4, _I64),
    "nt_beam_select": ([_I32] + [_I64] * 4 + [_P, _I64, _P, _P, _P, ctypes.c_double, _I64, _I32] + [_P] * 4 + [_I64, _P], _I32),
    "nt_reorder_rows": ([_I64, _P, _I64, _I64, _P, _P], _I32),
    "nt_kv_fork_workspace_bytes": ([_I64] * 3, _I64),
    "nt_kv_fork": ([_I64] * 7 + [_P, _I64] + [_P] * 6 + [_I64, _P], _I32),
    "nt_kv_copy_pages": ([_I64, _P] + [_I64] * 5 + [_P, _P], _I32),
    "nt_kv_attention_shared_workspace_bytes": ([_I32] + [_I64] * 9, _I64),
    "nt_kv_attention_shared": ([_I32] + [_I64] * 10 + [_F32, _P, _I64, _I64, _I64] + [_P] * 5 + [_I64] + [_P] * 5 + [_I64, _P], _I32),
    "nt_call_packed": ([_I32, ctypes.c_char_p, _I64], _I32),
}

EXPORTED = tuple(_SIGS)


def library_path() -> str:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Load the shared library once (raises NativeError when it is missing)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(_LIB_PATH):
                raise NativeError("load", 4, f"{_LIB_PATH} is missing; build it with "
                                  "`python -m neuratensor_b200.build`")
            lib = ctypes.CDLL(_LIB_PATH)
            for name, (args, res) in _SIGS.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = res
            _lib = lib
    return _lib


def _check(fn: str, rc: int) -> None:
    if rc != 0:
        msg = load().nt_last_error().decode(errors="replace")
        raise NativeError(fn, rc, msg)


def _p(t: Optional[Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(dev: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


_checked_devices = set()


def _device_index(*ts: Optional[Tensor]) -> int:
    """The CUDA device that all of `ts` are on."""
    idx = None
    for t in ts:
        if t is not None:
            i = t.get_device()                    # -1 for a CPU tensor
            if i != idx:
                if i < 0 or not t.is_cuda:
                    raise RuntimeError("neuratensor_b200 runs its hot path on CUDA (sm_100 / B200) only; "
                                       f"got a tensor on {t.device}")
                if idx is not None:
                    raise RuntimeError(f"tensors on different devices: cuda:{idx} and {t.device}")
                idx = i
    if idx is None:
        raise RuntimeError("no CUDA tensor given")
    if idx not in _checked_devices:
        _check("nt_device_supported", load().nt_device_supported(idx))
        _checked_devices.add(idx)
    return idx


def _require_cuda(*ts: Optional[Tensor]) -> torch.device:
    return torch.device("cuda", _device_index(*ts))


def _dtype_code(t: Tensor) -> int:
    if t.dtype not in _DT:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32 or bfloat16")
    return _DT[t.dtype]


def _workspace(nbytes: int, dev) -> Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=dev)


def _c(t: Optional[Tensor], dtype=None) -> Optional[Tensor]:
    if t is None:
        return None
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t.contiguous()


# --------------------------------------------------------------------------- #
#  Entry points                                                                #
# --------------------------------------------------------------------------- #

def lif_scan(x: Tensor, beta: Tensor, threshold: Tensor, membrane: Optional[Tensor] = None,
             spike_count: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """LIFLayer.forward (snn.py:264-312): x [B,T,C] -> (spikes [B,T,C], membrane [B,C])."""
    dev = _require_cuda(x, beta, threshold, membrane)
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, C], got {tuple(x.shape)}")
    B, T, C = x.shape
    if x.stride(2) != 1:
        x = x.contiguous()
    dt = x.dtype
    beta, threshold = _c(beta, dt), _c(threshold, dt)
    if beta.numel() != C or threshold.numel() != C:
        raise ValueError("beta / threshold must have C elements")
    mem_in = None if membrane is None else _c(membrane, dt)
    if mem_in is not None and mem_in.shape != (B, C):
        raise ValueError(f"membrane must be [B, C] = {(B, C)}, got {tuple(mem_in.shape)}")
    spikes = torch.empty((B, T, C), dtype=dt, device=dev)
    mem_out = torch.empty((B, C), dtype=dt, device=dev)
    rc = load().nt_lif_scan(_dtype_code(x), B, T, C, _p(x), x.stride(0), x.stride(1), _p(beta), _p(threshold),
                            _p(mem_in), _p(mem_out), _p(spikes), spikes.stride(0), spikes.stride(1),
                            _p(spike_count), _stream(dev))
    _check("nt_lif_scan", rc)
    return spikes, mem_out


def selective_scan(u: Tensor, dt: Tensor, Bm: Tensor, Cm: Tensor, log_A: Tensor, D: Tensor,
                   state: Optional[Tensor] = None, gate: Optional[Tensor] = None,
                   state_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """_discretize + _scan_sequential (ssm.py:106-139,184-221) -> (y [B,T,d], state [B,d,N])."""
    dev = _require_cuda(u, dt, Bm, Cm, log_A, D, state, gate)
    a = u.dtype
    B, T, d = u.shape
    N = log_A.shape[-1]
    sdt = state_dtype or (state.dtype if state is not None else a)
    u, dt, Bm, Cm, log_A, D = (_c(t, a) for t in (u, dt, Bm, Cm, log_A, D))
    gate = _c(gate, a)
    st_in = _c(state, sdt)
    y = torch.empty((B, T, d), dtype=a, device=dev)
    st_out = torch.empty((B, d, N), dtype=sdt, device=dev)
    rc = load().nt_selective_scan(_dtype_code(u), _DT[sdt], B, T, d, N, _p(u), _p(dt), _p(Bm), _p(Cm), _p(log_A),
                                  _p(D), _p(gate), _p(st_in), _p(st_out), _p(y), _stream(dev))
    _check("nt_selective_scan", rc)
    return y, st_out


def ssm_forward(u: Tensor, W_proj: Tensor, b_dt: Tensor, log_A: Tensor, D: Tensor,
                state: Optional[Tensor] = None, state_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """SelectiveSSMLayer.forward (ssm.py:313-349) with the packed [W_dt; W_B; W_C] weight."""
    dev = _require_cuda(u, W_proj, b_dt, log_A, D, state)
    a = u.dtype
    B, T, d = u.shape
    N = log_A.shape[-1]
    sdt = state_dtype or (state.dtype if state is not None else a)
    u = _c(u)
    st_in = _c(state, sdt)
    y = torch.empty((B, T, d), dtype=a, device=dev)
    st_out = torch.empty((B, d, N), dtype=sdt, device=dev)
    L = load()
    nbytes = L.nt_ssm_workspace_bytes(_DT[a], B, T, d, N)
    ws = _workspace(nbytes, dev)
    rc = L.nt_ssm_forward(_DT[a], _DT[sdt], B, T, d, N, _p(u), _p(W_proj), _p(b_dt), _p(log_A), _p(D), _p(st_in),
                          _p(st_out), _p(y), _p(ws), nbytes, _stream(dev))
    _check("nt_ssm_forward", rc)
    return y, st_out


def sparse_out_proj(o: Tensor, spikes: Tensor, W: Tensor) -> Tuple[Tensor, Tensor]:
    """_sparse_out_proj (fused.py:149-165): returns (out, n_active as a device int64 tensor)."""
    dev = _require_cuda(o, spikes, W)
    a = o.dtype
    lead = o.shape[:-1]
    K = o.shape[-1]
    M = o.numel() // K
    Nout = W.shape[0]
    o2, s2, W2 = _c(o), _c(spikes, a), _c(W, a)
    out = torch.empty((*lead, Nout), dtype=a, device=dev)
    n_active = torch.empty((), dtype=torch.int64, device=dev)
    L = load()
    nbytes = L.nt_sparse_out_proj_workspace_bytes(_DT[a], M, K, Nout)
    ws = _workspace(nbytes, dev)
    rc = L.nt_sparse_out_proj(_DT[a], M, K, Nout, _p(o2), _p(s2), _p(W2), _p(out), _p(n_active), _p(ws), nbytes,
                              _stream(dev))
    _check("nt_sparse_out_proj", rc)
    return out, n_active


def rmsnorm_in_proj(x: Tensor, gamma: Tensor, W_in: Tensor) -> Tuple[Tensor, Tensor]:
    """norm + in_proj + chunk (fused.py:118-119): x [..., dm] -> (h, gate) [..., di]."""
    dev = _require_cuda(x, gamma, W_in)
    a = x.dtype
    dm = x.shape[-1]
    di = W_in.shape[0] // 2
    M = x.numel() // dm
    x2, g2, W2 = _c(x), _c(gamma, a), _c(W_in, a)
    h = torch.empty((*x.shape[:-1], di), dtype=a, device=dev)
    gate = torch.empty_like(h)
    L = load()
    nbytes = L.nt_rmsnorm_in_proj_workspace_bytes(_DT[a], M, dm, di)
    ws = _workspace(nbytes, dev)
    rc = L.nt_rmsnorm_in_proj(_DT[a], M, dm, di, _p(x2), _p(g2), _p(W2), _p(h), _p(gate), _p(ws), nbytes,
                              _stream(dev))
    _check("nt_rmsnorm_in_proj", rc)
    return h, gate


def rmsnorm_in_proj_noalloc(x: Tensor, gamma: Tensor, W_in: Tensor) -> Tuple[Tensor, Tensor]:
    """rmsnorm_in_proj without a workspace: for callers that cannot allocate device
    memory at call time; the library's own static scratch holds the normalised rows
    (at most nt_noalloc_scratch_bytes() of them).  Calls overlapping on the GPU race."""
    dev = _require_cuda(x, gamma, W_in)
    a = x.dtype
    dm = x.shape[-1]
    di = W_in.shape[0] // 2
    M = x.numel() // dm
    x2, g2, W2 = _c(x), _c(gamma, a), _c(W_in, a)
    h = torch.empty((*x.shape[:-1], di), dtype=a, device=dev)
    gate = torch.empty_like(h)
    rc = load().nt_rmsnorm_in_proj_noalloc(_DT[a], M, dm, di, _p(x2), _p(g2), _p(W2), _p(h), _p(gate), _stream(dev))
    _check("nt_rmsnorm_in_proj_noalloc", rc)
    return h, gate


def block_forward(x: Tensor, norm_w: Tensor, W_in: Tensor, beta: Tensor, threshold: Tensor, log_A: Tensor,
                  D: Tensor, W_proj: Tensor, b_dt: Tensor, W_out: Tensor, out_scale: Tensor,
                  membrane: Optional[Tensor], ssm_state: Optional[Tensor], spike_count: Tensor,
                  sparse: bool = True, state_dtype: Optional[torch.dtype] = None,
                  workspace: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """FusedSpikeBlock.forward (fused.py:101-147) -> (out, membrane, ssm_state).

    All weight tensors must already be contiguous and in x.dtype; spike_count
    is a device int64 scalar incremented by the block's spike count.
    """
    dev = x.device
    a = x.dtype
    B, T, dm = x.shape
    di = W_in.shape[0] // 2
    N = log_A.shape[-1]
    sdt = state_dtype or a
    x = x.contiguous()
    mem_in = None if membrane is None else _c(membrane, a)
    st_in = None if ssm_state is None else _c(ssm_state, sdt)
    out = torch.empty_like(x)
    mem_out = torch.empty((B, di), dtype=a, device=dev)
    st_out = torch.empty((B, di, N), dtype=sdt, device=dev)
    L = load()
    nbytes = L.nt_block_workspace_bytes(_DT[a], B, T, dm, di, N)
    ws = workspace if (workspace is not None and workspace.numel() >= nbytes) else _workspace(nbytes, dev)
    rc = L.nt_block_forward(_DT[a], _DT[sdt], B, T, dm, di, N, _p(x), _p(norm_w), _p(W_in), _p(beta), _p(threshold),
                            _p(log_A), _p(D), _p(W_proj), _p(b_dt), _p(W_out), _p(out_scale), _p(mem_in),
                            _p(mem_out), _p(st_in), _p(st_out), _p(out), _p(spike_count), 1 if sparse else 0,
                            _p(ws), ws.numel(), _stream(dev))
    _check("nt_block_forward", rc)
    return out, mem_out, st_out


def block_workspace_bytes(dtype: torch.dtype, B: int, T: int, dm: int, di: int, N: int) -> int:
    return int(load().nt_block_workspace_bytes(_DT[dtype], B, T, dm, di, N))


def lif_ssm_fused(x: Tensor, delta: Tensor, Bm: Tensor, Cm: Tensor, log_A: Tensor, Dskip: Tensor, beta: Tensor,
                  threshold: Tensor, membrane: Optional[Tensor] = None, state: Optional[Tensor] = None,
                  spike_dtype: Optional[torch.dtype] = torch.uint8, spike_count: Optional[Tensor] = None):
    """LIF spikes of x driving the selective scan with given dt/B/C (bf16 activations, fp32 state).

    Returns (y [B,L,d] bf16, spikes [B,L,d] or None, membrane [B,d] f32, state [B,d,N] f32).
    """
    dev = _require_cuda(x, delta, Bm, Cm, log_A, Dskip, beta, threshold, membrane, state)
    B, L_, d = x.shape
    N = log_A.shape[-1]
    bf = torch.bfloat16
    x, delta, Bm, Cm = (_c(t, bf) for t in (x, delta, Bm, Cm))
    log_A, Dskip, beta, threshold = (_c(t, torch.float32) for t in (log_A, Dskip, beta, threshold))
    mem_in = _c(membrane, torch.float32)
    st_in = _c(state, torch.float32)
    y = torch.empty((B, L_, d), dtype=bf, device=dev)
    spikes = None if spike_dtype is None else torch.empty((B, L_, d), dtype=spike_dtype, device=dev)
    sd = {torch.uint8: NT_U8, torch.bfloat16: NT_BF16, None: NT_U8}[spike_dtype]
    mem_out = torch.empty((B, d), dtype=torch.float32, device=dev)
    st_out = torch.empty((B, d, N), dtype=torch.float32, device=dev)
    rc = load().nt_lif_ssm_fused(B, L_, d, N, _p(x), _p(delta), _p(Bm), _p(Cm), _p(log_A), _p(Dskip), _p(beta),
                                 _p(threshold), _p(mem_in), _p(mem_out), _p(st_in), _p(st_out), _p(y), _p(spikes),
                                 sd, _p(spike_count), _stream(dev))
    _check("nt_lif_ssm_fused", rc)
    return y, spikes, mem_out, st_out


def window_attention(qkv: Tensor, n_heads: int, window: int, cos: Tensor, sin: Tensor) -> Tensor:
    """RoPE + sliding-window causal SDPA of SlidingWindowAttention.forward (model.py:159-178).

    qkv: [B, T, 3*d_model] bf16 (the qkv projection's output), head_dim =
    d_model / n_heads of 64 or 128; cos/sin: [T, head_dim] rotary tables;
    returns the attention output [B, T, d_model] (heads concatenated, as
    o_proj takes it)."""
    dev = _require_cuda(qkv, cos, sin)
    if qkv.dtype != torch.bfloat16:
        raise NativeError("nt_window_attention", 2, "bf16 only")
    if qkv.dim() != 3:
        raise ValueError(f"qkv must be [B, T, 3*d_model], got {tuple(qkv.shape)}")
    B, T, three_dm = qkv.shape
    dm = three_dm // 3
    hd = dm // n_heads if n_heads > 0 else 0
    if three_dm != 3 * dm or hd not in (64, 128) or dm != hd * n_heads:
        raise ValueError(f"qkv width {three_dm} does not split into {n_heads} heads of 64 or 128")
    if qkv.stride(2) != 1 or qkv.stride(0) != T * qkv.stride(1):
        qkv = qkv.contiguous()
    cos = cos[:T].to(torch.bfloat16).contiguous()
    sin = sin[:T].to(torch.bfloat16).contiguous()
    if cos.shape != (T, hd) or sin.shape != (T, hd):
        raise ValueError(f"cos/sin must hold at least T rows of {hd}")
    out = torch.empty((B, T, dm), dtype=torch.bfloat16, device=dev)
    rc = load().nt_window_attention(_dtype_code(qkv), B, T, n_heads, hd, int(window), _p(qkv), qkv.stride(1),
                                    _p(cos), _p(sin), _p(out), out.stride(1), _stream(dev))
    _check("nt_window_attention", rc)
    return out


def attention_forward(x: Tensor, norm_w: Tensor, W_qkv: Tensor, W_o: Tensor, n_heads: int, window: int,
                      cos: Tensor, sin: Tensor, workspace: Optional[Tensor] = None) -> Tensor:
    """SlidingWindowAttention.forward (model.py:148-181) in one call: RMSNorm, qkv
    projection, RoPE + windowed causal attention, o_proj + residual.  bf16, head_dim 64 or 128."""
    dev = _require_cuda(x, norm_w, W_qkv, W_o, cos, sin)
    if x.dtype != torch.bfloat16:
        raise NativeError("nt_attention_forward", 2, "bf16 only")
    B, T, dm = x.shape
    hd = dm // n_heads
    x = x.contiguous()
    nw, Wq, Wo = _c(norm_w, x.dtype), _c(W_qkv, x.dtype), _c(W_o, x.dtype)
    cos = cos[:T].to(torch.bfloat16).contiguous()
    sin = sin[:T].to(torch.bfloat16).contiguous()
    if cos.shape != (T, hd) or sin.shape != (T, hd):
        raise ValueError(f"cos/sin must hold at least T rows of {hd}")
    out = torch.empty_like(x)
    L = load()
    nbytes = L.nt_attention_workspace_bytes(_DT[x.dtype], B, T, dm)
    ws = workspace if (workspace is not None and workspace.numel() >= nbytes) else _workspace(nbytes, dev)
    rc = L.nt_attention_forward(_DT[x.dtype], B, T, dm, n_heads, int(window), _p(x), _p(nw), _p(Wq), _p(Wo),
                                _p(cos), _p(sin), _p(out), _p(ws), ws.numel(), _stream(dev))
    _check("nt_attention_forward", rc)
    return out


def attention_output(o: Tensor, W_o: Tensor, x: Tensor) -> Tensor:
    """o_proj + residual (model.py:180-181), the end of attention_forward for attention that
    was taken elsewhere: o [..., d_model] @ W_o^T, rounded, + x in x.dtype."""
    dev = _require_cuda(o, W_o, x)
    if o.shape != x.shape or o.dtype != x.dtype or W_o.shape != (x.shape[-1], x.shape[-1]):
        raise ValueError(f"o and x must be [..., d_model] of one dtype and W_o [d_model, d_model], got {tuple(o.shape)} "
                         f"{o.dtype}, {tuple(x.shape)} {x.dtype} and {tuple(W_o.shape)}")
    dm = x.shape[-1]
    o, W, x = _c(o), _c(W_o, x.dtype), _c(x)
    out = torch.empty_like(x)
    rc = load().nt_attention_output(_dtype_code(x), x.numel() // dm, dm, _p(o), _p(W), _p(x), _p(out), _stream(dev))
    _check("nt_attention_output", rc)
    return out


def greedy_tokens(logits: Tensor, u: Tensor, out: Optional[Tensor] = None) -> Tensor:
    """top_k = 1 sampling of generate (model.py:344-359): per row of logits [B, V],
    uniformly among the entries equal to the row maximum, chosen by u [B] in [0, 1).
    Returns int64 tokens [B, 1] (written into `out` when given)."""
    dev = _require_cuda(logits, u)
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be [B, V] with unit column stride")
    B, V = logits.shape
    u = _c(u, torch.float32)
    if out is None:
        out = torch.empty((B, 1), dtype=torch.int64, device=dev)
    rc = load().nt_greedy_tokens(_dtype_code(logits), B, V, _p(logits), logits.stride(0), _p(u), _p(out),
                                 _stream(dev))
    _check("nt_greedy_tokens", rc)
    return out


def embedding(ids: Tensor, W: Tensor) -> Tensor:
    """nn.Embedding lookup (model.py:258): ids [...] int64 -> [..., d_model] in W's dtype.
    An id outside [0, vocab) gives a zero row and a flag in the device error word."""
    dev = _require_cuda(ids, W)
    W = _c(W)
    ids = ids.to(torch.int64).contiguous()
    vocab, dm = W.shape
    out = torch.empty((*ids.shape, dm), dtype=W.dtype, device=dev)
    rc = load().nt_embedding(_dtype_code(W), ids.numel(), dm, vocab, _p(ids), _p(W), _p(out), _stream(dev))
    _check("nt_embedding", rc)
    return out


def lm_head(x: Tensor, gamma: Tensor, W: Tensor, workspace: Optional[Tensor] = None,
            out: Optional[Tensor] = None) -> Tensor:
    """Final RMSNorm + tied lm_head (model.py:283-284): x [..., dm] -> logits [..., vocab] in x.dtype
    (written into `out`, a contiguous tensor of that shape, when given)."""
    dev = _require_cuda(x, gamma, W)
    a = x.dtype
    dm = x.shape[-1]
    vocab = W.shape[0]
    M = x.numel() // dm
    x2, g2, W2 = _c(x), _c(gamma, a), _c(W, a)
    if out is not None:
        if out.dtype != a or not out.is_contiguous() or out.numel() != M * vocab:
            raise ValueError("out must be a contiguous [..., vocab] tensor in x.dtype")
        logits = out
    else:
        logits = torch.empty((*x.shape[:-1], vocab), dtype=a, device=dev)
    L = load()
    nbytes = L.nt_lm_head_workspace_bytes(_DT[a], M, dm, vocab)
    ws = workspace if (workspace is not None and workspace.numel() >= nbytes) else _workspace(nbytes, dev)
    rc = L.nt_lm_head(_DT[a], M, dm, vocab, _p(x2), _p(g2), _p(W2), _p(logits), _p(ws), ws.numel(), _stream(dev))
    _check("nt_lm_head", rc)
    return logits


# --------------------------------------------------------------------------- #
#  A generation step with an attention memory: rotary positions, the 8-bit     #
#  cache, attention over it, penalties on logits                               #
# --------------------------------------------------------------------------- #

# entry point -> (its number, number of arguments, packer) for nt_call_packed
_PACKED = {"nt_rotary": (0, 21, struct.Struct("=8qd12q").pack), "nt_kv_append": (1, 25, struct.Struct("=25q").pack),
           "nt_kv_attention": (2, 27, struct.Struct("=10qd16q").pack),
           "nt_logits_process": (3, 27, struct.Struct("=11qqdqdqd10q").pack),
           "nt_beam_select": (4, 19, struct.Struct("=10qd8q").pack), "nt_reorder_rows": (5, 6, struct.Struct("=6q").pack),
           "nt_kv_fork": (6, 17, struct.Struct("=17q").pack), "nt_kv_copy_pages": (7, 9, struct.Struct("=9q").pack),
           "nt_kv_attention_shared": (8, 29, struct.Struct("=11qd17q").pack)}


def _launch(index: int, name: str, *args) -> None:
    """Calls an entry point with device `index` current and its current stream as the last argument.

    These calls are short (a step makes several per layer), so their arguments go over in
    one piece, the stream is read as the raw handle and the device switched only when it has to be."""
    entry, n, pack = _PACKED[name]
    words = pack(*args, torch._C._cuda_getCurrentRawStream(index))
    if index == torch._C._cuda_getDevice():
        rc = _lib.nt_call_packed(entry, words, n)
    else:
        with torch.cuda.device(index):
            rc = _lib.nt_call_packed(entry, words, n)
    if rc != 0:
        _check(name, rc)


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _like(t: Tensor) -> Tensor:
    """An uninitialised contiguous tensor of t's shape, dtype and device."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _has_tangent(*ts: Optional[Tensor]) -> bool:
    """Whether one of `ts` carries a forward-mode derivative (the level is -1 where there can be none)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _refuse_grad(fn: str, *ts: Optional[Tensor]) -> None:
    for t in ts:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{fn} has no backward; detach the inputs or run under torch.no_grad()")
    if _has_tangent(*ts):
        raise RuntimeError(f"{fn} has no derivative in forward mode; take the primal of the inputs")


def _refuse_out(fn: str, *ts: Tensor) -> None:
    """What is written must not be part of a graph, as for torch's own out= and in-place operations."""
    for t in ts:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{fn} writes a tensor that requires grad; detach it or run under torch.no_grad()")
    if _has_tangent(*ts):
        raise RuntimeError(f"{fn} writes a tensor with a forward-mode derivative, which would stay as it was")


def _ints(t: Tensor, dtype: torch.dtype, what: str) -> Tensor:
    if t.dtype == dtype:
        return t
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
    return t.to(dtype)


def _indexes(t: Tensor, what: str) -> Tensor:
    """_ints as int32, in which what does not fit stays out of range (6 us more for int64, a launch)."""
    if t.dtype == torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return _ints(t, torch.int32, what)


class _Rotary(torch.autograd.Function):
    # forward takes ctx: with the separate setup_context that torch.func asks for, a pass of both directions that
    # is waited for takes 328 us where it takes 307 (32767 tokens of 24 float32 heads), so torch.func is refused
    @staticmethod
    def forward(ctx, x, positions, inv_freq, layout, mscale, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.how = (layout, mscale, inverse)
        return _rotary(x, positions, inv_freq, layout, mscale, inverse, None)

    @staticmethod
    def backward(ctx, g):
        positions, inv_freq = ctx.saved_tensors
        layout, mscale, inverse = ctx.how
        return rotary(g, positions, inv_freq, layout, mscale, not inverse), None, None, None, None, None

    @staticmethod
    def jvp(ctx, t, *_):                    # linear in x: the tangent turns as x does
        return rotary(t, *ctx.saved_tensors, *ctx.how)


def rotary(x: Tensor, positions: Tensor, inv_freq: Tensor, layout: str = "half", mscale: float = 1.0,
           inverse: bool = False, out: Optional[Tensor] = None) -> Tensor:
    """Rotary positions (the rotation of apply_rotary, model.py:119-126, at any positions).

    x: [B, T, H, D] float32 or bfloat16, any strides with unit stride in D (q|k of a qkv
    projection can be rotated where they lie); positions: int64 [B, T], or [T] for all
    rows; inv_freq: [R/2] float32, the first R <= D dimensions turn and the rest are
    copied.  layout "half" pairs (i, i + R/2), "interleaved" (2i, 2i + 1).  Pair i turns
    by positions * inv_freq[i], taken in float64, and is multiplied by mscale; one
    rounding.  inverse turns backwards.  out may be x (in place), or must not overlap it.
    Differentiable in x (not with out), forwards and backwards.  Heads of at most 2048 dimensions."""
    if (x.requires_grad or inv_freq.requires_grad) and torch.is_grad_enabled() or _has_tangent(x, inv_freq):
        if inv_freq.requires_grad and torch.is_grad_enabled() or _has_tangent(inv_freq):
            raise RuntimeError("rotary has no gradient for inv_freq; detach it")
        if out is not None:
            raise RuntimeError("rotary with out= has no backward; detach x or leave out away")
        return _Rotary.apply(x, positions, inv_freq, layout, mscale, inverse)
    return _rotary(x, positions, inv_freq, layout, mscale, inverse, out)


def _rotary(x, positions, inv_freq, layout, mscale, inverse, out):
    index = _device_index(x, positions, inv_freq, out)
    code = _dtype_code(x)
    if x.dim() != 4:
        raise ValueError(f"x must be [B, T, H, D], got {tuple(x.shape)}")
    B, T, H, D = x.shape
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a float32 vector of R/2 frequencies")
    R = 2 * inv_freq.numel()
    if not 2 <= R <= D:
        raise ValueError(f"{R} rotated dimensions do not fit a head of {D}")
    if positions.dtype != torch.int64:
        positions = _ints(positions, torch.int64, "positions")
    if positions.shape != (B, T):
        if positions.dim() not in (1, 2) or positions.shape[-1] != T:
            raise ValueError(f"positions must be [T] or [B, T] = {(B, T)}, got {tuple(positions.shape)}")
        positions = positions.expand(B, T)
    p_sb, p_st = positions.stride()
    if p_st != 1 and T > 1:
        positions = positions.contiguous()
        p_sb = T
    x_sb, x_st, x_sh, unit = x.stride()
    if unit != 1 and D > 1:
        x = x.contiguous()
        x_sb, x_st, x_sh, _ = x.stride()
    given = out is not None
    if not given:
        out = _like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.stride(3) != 1:
        raise ValueError("out must have x's shape and dtype and unit stride in D")
    elif any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError("out must not overlap itself")
    else:
        _refuse_out("rotary", out)
    y_sb, y_st, y_sh, _ = out.stride()
    inv_freq = inv_freq.contiguous()
    _launch(index, "nt_rotary", code, B, T, H, D, R, layout == "interleaved", inverse, mscale, x.data_ptr(), x_sb, x_st, x_sh,
            positions.data_ptr(), p_sb, inv_freq.data_ptr(), out.data_ptr(), y_sb, y_st, y_sh)
    if given:
        increment_version(out)          # so that a backward pass that saved it before knows
    return out


def _row_ints(fn: str, what: str, t: Optional[Tensor], B: int) -> Optional[Tensor]:
    """An integer per row as contiguous int32 [B]."""
    if t is None:
        return None
    if t.shape != (B,):
        raise ValueError(f"{fn}: {what} must be [{B}], got {tuple(t.shape)}")
    if t.dtype != torch.int32:
        t = _ints(t, torch.int32, what)
    return t.contiguous()


def _cache_args(fn, B, D, k_codes, k_scale, v_codes, v_scale, table, lengths, counts):
    """Checks the tensors of a cache; returns (heads, page, pages, blocks, table, lengths, counts)."""
    shape = k_codes.shape
    if len(shape) != 4 or v_codes.shape != shape or shape[3] != D:
        raise ValueError(f"{fn}: codes must be [pages, heads, page, {D}], got {tuple(shape)} and {tuple(v_codes.shape)}")
    for t in (k_codes, v_codes):
        dtype = t.dtype
        if dtype != torch.float8_e4m3fn and dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"{fn}: codes must be contiguous float8_e4m3fn (or its bytes as uint8)")
    n, H, P, _ = shape
    per_head = (n, H)
    for t in (k_scale, v_scale):
        if t.dtype != torch.float32 or t.shape != per_head or not t.is_contiguous():
            raise ValueError(f"{fn}: scales must be contiguous float32 [pages, heads] = {per_head}")
    entries = table.shape
    if table.dtype != torch.int32 or len(entries) != 2 or entries[0] != B or (entries[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{fn}: table must be int32 [{B}, blocks] with unit stride")
    return H, P, n, entries[1], _row_ints(fn, "lengths", lengths, B), _row_ints(fn, "counts", counts, B)


def kv_append(k: Tensor, v: Tensor, k_codes: Tensor, k_scale: Tensor, v_codes: Tensor, v_scale: Tensor, table: Tensor,
              lengths: Tensor, counts: Optional[Tensor] = None) -> None:
    """Writes new keys and values into the paged 8-bit cache, in place.

    k, v: [B, T, H, D] float32 or bfloat16 (unit stride in D, D 64 or 128); codes:
    [pages, H, page, D] float8_e4m3fn, page 16, 32 or 64; scales: [pages, H] float32, one
    power of two per page and head; table: int32 [B, blocks], position p of sequence b
    lies in page table[b, p // page].  lengths [B]: tokens of each sequence with the new
    ones; counts [B] (None: T): how many of the T rows are new, rows 0..counts-1, which
    become the last counts positions.  A page's scale grows with its largest value, and
    its older codes are re-encoded then.  A page that is written must belong to one
    sequence and stand once among its blocks; a bad length, count or page is skipped and
    flagged (device_error_flags)."""
    _refuse_grad("kv_append", k, v)
    _refuse_out("kv_append", k_codes, k_scale, v_codes, v_scale)
    index = _device_index(k, v, k_codes, k_scale, v_codes, v_scale, table, lengths, counts)
    code = _dtype_code(k)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must be [B, T, H, D] of one dtype, got {tuple(shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    B, T, H, D = shape
    heads, P, n, blocks, lengths, counts = _cache_args("kv_append", B, D, k_codes, k_scale, v_codes, v_scale, table,
                                                       lengths, counts)
    if heads != H:
        raise ValueError(f"kv_append: the cache has {heads} heads, k and v have {H}")
    if k_codes.data_ptr() == v_codes.data_ptr() and n:
        raise ValueError("kv_append: keys and values need a cache each")
    k_sb, k_st, k_sh, unit = k.stride()
    if unit != 1:
        k = k.contiguous()
        k_sb, k_st, k_sh, _ = k.stride()
    v_sb, v_st, v_sh, unit = v.stride()
    if unit != 1:
        v = v.contiguous()
        v_sb, v_st, v_sh, _ = v.stride()
    _launch(index, "nt_kv_append", code, B, T, H, D, P, n, blocks, k.data_ptr(), k_sb, k_st, k_sh, v.data_ptr(), v_sb, v_st,
            v_sh, k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(), table.data_ptr(),
            table.stride(0), lengths.data_ptr(), _ptr(counts))
    increment_version((k_codes, k_scale, v_codes, v_scale))


@functools.lru_cache(maxsize=256)
def _kv_attention_bytes(*sizes: int) -> int:
    return load().nt_kv_attention_workspace_bytes(*sizes)


def kv_attention(q: Tensor, k_codes: Tensor, k_scale: Tensor, v_codes: Tensor, v_scale: Tensor, table: Tensor,
                 lengths: Tensor, counts: Optional[Tensor] = None, window: Optional[int] = None,
                 scale: Optional[float] = None) -> Tensor:
    """Attention of the new tokens over the paged 8-bit cache (kv_append) -> [B, T, Hq, D].

    q: [B, T, Hq, D] float32 or bfloat16, Hq a multiple of the cache's heads; row
    t < counts[b] stands at lengths[b] - counts[b] + t and sees the keys up to it, with a
    window only those from position - window on.  Other rows are zero.  scale: of the
    scores, 1/sqrt(D) by default."""
    _refuse_grad("kv_attention", q, k_codes, k_scale, v_codes, v_scale)
    index = _device_index(q, k_codes, k_scale, v_codes, v_scale, table, lengths, counts)
    code = _dtype_code(q)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, T, H, D], got {tuple(q.shape)}")
    B, T, Hq, D = q.shape
    H, P, n, blocks, lengths, counts = _cache_args("kv_attention", B, D, k_codes, k_scale, v_codes, v_scale, table,
                                                   lengths, counts)
    if H < 1 or Hq < H or Hq % H:
        raise ValueError(f"kv_attention: {Hq} query heads over {H} cached heads")
    if window is not None and window < 0:
        raise ValueError(f"kv_attention: window must be None or >= 0, got {window}")
    win = -1 if window is None else min(int(window), 2 ** 31)      # as good as none from there on
    if q.stride(3) != 1:
        q = q.contiguous()
    q_sb, q_st, q_sh, _ = q.stride()
    out = _like(q)
    nbytes = _kv_attention_bytes(B, T, Hq, H, D, P, blocks, win)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(index, "nt_kv_attention", code, B, T, Hq, H, D, P, n, blocks, win, D ** -0.5 if scale is None else scale,
            q.data_ptr(), q_sb, q_st, q_sh, k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(),
            table.data_ptr(), table.stride(0), lengths.data_ptr(), _ptr(counts), out.data_ptr(), _ptr(ws), nbytes)
    return out


def _per_row(name: str, v, B: int, none: float, index: int) -> Tuple[Optional[Tensor], float]:
    """A penalty as ([B] float32, unused) or (None, scalar)."""
    if v is None:
        return None, none
    if isinstance(v, Tensor):
        if v.shape != (B,):
            raise ValueError(f"{name} must be a number or [{B}], got {tuple(v.shape)}")
        if v.get_device() != index:
            raise RuntimeError(f"{name} must be on CUDA device {index}, got {v.device}")
        return _c(v, torch.float32), none
    return None, float(v)


def logits_process(logits: Tensor, tokens: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                   prompt_lengths: Optional[Tensor] = None, repetition: Union[None, float, Tensor] = None,
                   frequency: Union[None, float, Tensor] = None, presence: Union[None, float, Tensor] = None,
                   each: bool = False, bias_ids: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                   allowed: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """Penalties for repeated tokens, biases and masks on logits [B, V], one pass (model.py:336-342 and more).

    tokens: [B, L] int64 history, of which row b counts the first lengths[b] (None: L); ids
    outside the vocabulary are skipped.  repetition r (a number or [B]): a logit x whose
    token is in the history becomes x / r if positive, else x * r; with each=True once per
    occurrence, rounded each time, as generate does.  frequency and presence: what is
    taken off per occurrence and for any, counted from prompt_lengths[b] (None: 0) on.
    bias_ids [B, N] int64 and bias [B, N]: added to the logits of the ids (-1: none; of
    equal ids the last holds).  allowed: int32 words [B or 1, ceil(V / 32)]; a zero bit v % 32 of
    word v // 32 makes the logit -inf (pack_allowed), all of a row without a bit: it has no
    probabilities, so ask for them only where a token is left.  float32 arithmetic, one
    rounding; out may be logits."""
    index = _device_index(logits, tokens, lengths, prompt_lengths, bias_ids, bias, allowed, out)
    code = _dtype_code(logits)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    L = tok_ld = 0
    if tokens is not None:
        tokens = _ints(tokens, torch.int64, "tokens")
        if tokens.dim() != 2 or tokens.shape[0] != B:
            raise ValueError(f"tokens must be [{B}, L], got {tuple(tokens.shape)}")
        L = tokens.shape[1]
        if L > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        tok_ld = tokens.stride(0)
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths of a history that is not given")
    lengths = _row_ints("logits_process", "lengths", lengths, B)
    prompt_lengths = _row_ints("logits_process", "prompt_lengths", prompt_lengths, B)
    if each and prompt_lengths is not None:
        raise ValueError("a repetition penalty per occurrence takes no prompt_lengths")
    rep, rep_all = _per_row("repetition", repetition, B, 1.0, index)
    fq, fq_all = _per_row("frequency", frequency, B, 0.0, index)
    ps, ps_all = _per_row("presence", presence, B, 0.0, index)
    _refuse_grad("logits_process", logits, bias, rep, fq, ps)
    if rep is None and not (math.isfinite(rep_all) and (rep_all > 0.0 or each and rep_all != 0.0)):
        raise ValueError(f"repetition must be {'finite and not' if each else 'above'} 0, got {rep_all}")
    NB = ids_ld = bias_ld = 0
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias_ids is not None:
        if bias_ids.dim() != 2 or bias_ids.shape[0] != B or bias.shape != bias_ids.shape:
            raise ValueError(f"bias_ids and bias must be [{B}, N], got {tuple(bias_ids.shape)} and {tuple(bias.shape)}")
        bias_ids = _ints(bias_ids, torch.int64, "bias_ids")
        bias = bias if bias.dtype == torch.float32 else bias.float()
        NB = bias.shape[1]
        if NB > 1 and bias_ids.stride(1) != 1:
            bias_ids = bias_ids.contiguous()
        if NB > 1 and bias.stride(1) != 1:
            bias = bias.contiguous()
        ids_ld, bias_ld = bias_ids.stride(0), bias.stride(0)
    allowed_ld = 0
    if allowed is not None:
        words = (V + 31) // 32
        if allowed.dtype not in (torch.int32, torch.uint32) or allowed.dim() != 2 or allowed.shape[0] not in (1, B) or \
                allowed.shape[1] < words:
            raise ValueError(f"allowed must be int32 [{B} or 1, {words}], got {allowed.dtype} {tuple(allowed.shape)}")
        if allowed.shape[1] > 1 and allowed.stride(1) != 1:
            allowed = allowed.contiguous()
        allowed_ld = allowed.stride(0) if allowed.shape[0] == B else 0
    given = out is not None
    if not given:
        out = _like(logits)
    elif out.shape != logits.shape or out.dtype != logits.dtype or (V > 1 and out.stride(1) != 1) or \
            (B > 1 and out.stride(0) < V):
        raise ValueError("out must be [B, V] in the logits' dtype with unit column stride")
    else:
        _refuse_out("logits_process", out)
    _launch(index, "nt_logits_process", code, B, V, logits.data_ptr(), logits.stride(0), _ptr(tokens), tok_ld, L,
            _ptr(lengths), _ptr(prompt_lengths), each, _ptr(rep), rep_all, _ptr(fq), fq_all, _ptr(ps), ps_all,
            _ptr(bias_ids), ids_ld, _ptr(bias), bias_ld, NB, _ptr(allowed), allowed_ld, out.data_ptr(), out.stride(0))
    if given:
        increment_version(out)
    return out


def pack_allowed(mask: Tensor) -> Tensor:
    """A boolean mask [B, V] of allowed tokens as the int32 words that logits_process takes."""
    if mask.dtype != torch.bool or mask.dim() != 2:
        raise ValueError("mask must be a boolean [B, V]")
    B, V = mask.shape
    bits = torch.zeros((B, (V + 31) // 32 * 32), dtype=torch.int64, device=mask.device)
    bits[:, :V] = mask
    words = (bits.view(B, -1, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


# --------------------------------------------------------------------------- #
#  A step of a beam search: the choice over beams and vocabulary, states moved #
#  to the chosen beams, pages of the cache forked, attention over shared ones  #
# --------------------------------------------------------------------------- #

@functools.lru_cache(maxsize=256)
def _beam_select_bytes(*sizes: int) -> int:
    return load().nt_beam_select_workspace_bytes(*sizes)


def beam_select(logits: Tensor, scores: Tensor, finished: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                length_penalty: float = 0.0, n: Optional[int] = None, pad: int = 0, stay: bool = False
                ) -> Tuple[Tensor, Tensor, Tensor]:
    """The best continuations of a beam search -> (scores [B, n], rows [B, n], tokens [B, n]).

    logits: [B*K, V] float32 or bfloat16, the K beams of an item after one another;
    scores: [B, K] float32, their log-probabilities so far.  A live beam offers every
    token whose logit is not -inf with its score and log-softmax added, a finished
    one (bool [B, K]) itself alone, with token `pad`; a beam with a score or a
    log-sum that is not finite offers nothing.  Candidates rank by that sum divided by
    the length to the power of length_penalty (lengths: [B, K], tokens made so
    far, one more for a live beam); ties go to the lower beam, then the lower token.  n
    (None: K; at most 64, like K) are wanted, best first; with stay, n is K and the
    best child of a beam stands in the beam's own place.  scores: float32 sums; rows:
    int32, the row of logits that each goes on from; tokens: int64.  Where candidates
    run out: -inf, row b*K + place % K, `pad`."""
    index = _device_index(logits, scores, finished, lengths)
    _refuse_grad("beam_select", logits, scores)
    code = _dtype_code(logits)
    if scores.dim() != 2 or scores.dtype != torch.float32 or scores.shape[1] < 1:
        raise ValueError(f"beam_select: scores must be float32 [B, K], got {scores.dtype} {tuple(scores.shape)}")
    B, K = scores.shape
    if logits.dim() != 2 or logits.shape[0] != B * K or logits.shape[1] < 1:
        raise ValueError(f"beam_select: logits must be [{B * K}, V], got {tuple(logits.shape)}")
    V = logits.shape[1]
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    if n is None:
        n = K
    if not 1 <= n <= 64 or K > 64:
        raise ValueError(f"beam_select: 1 to 64 beams and continuations, got {K} and {n}")
    if stay and n != K:
        raise ValueError(f"beam_select: children in their parents' places need n = K, got {n} of {K}")
    if finished is not None:
        if finished.shape != (B, K) or finished.dtype != torch.bool:
            raise ValueError(f"beam_select: finished must be bool [{B}, {K}], got {finished.dtype} {tuple(finished.shape)}")
        finished = finished.contiguous()
    if not math.isfinite(length_penalty):
        raise ValueError(f"beam_select: length_penalty must be finite, got {length_penalty}")
    if lengths is not None:
        if lengths.shape != (B, K):
            raise ValueError(f"beam_select: lengths must be [{B}, {K}], got {tuple(lengths.shape)}")
        lengths = _indexes(lengths, "lengths").contiguous()
    elif length_penalty != 0.0:
        raise ValueError("beam_select: a length penalty needs lengths")
    if not 0 <= pad < 2 ** 31:
        raise ValueError(f"beam_select: pad must be a token, got {pad}")
    scores = scores.contiguous()
    out = scores.new_empty((B, n))
    rows = torch.empty((B, n), dtype=torch.int32, device=scores.device)
    tokens = torch.empty((B, n), dtype=torch.int64, device=scores.device)
    nbytes = _beam_select_bytes(code, B, K, V, n)
    ws = scores.new_empty(max(nbytes, 1), dtype=torch.uint8)
    _launch(index, "nt_beam_select", code, B, K, V, n, logits.data_ptr(), logits.stride(0), scores.data_ptr(), _ptr(finished),
            _ptr(lengths), length_penalty, pad, stay, out.data_ptr(), rows.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes)
    return out, rows, tokens


def reorder_rows(tensors: Sequence[Tensor], rows: Tensor, group: Optional[int] = None) -> None:
    """Row r of every tensor takes what its row rows[r] held, in place and in one launch.

    tensors: any dtypes, [R, ...] with the same R and rows that lie in one piece (block
    states, for instance), not overlapping; rows: int32 or int64 [R], each within its group of
    `group` consecutive rows (None: R; at most 1024), -1: the row stays as it is.  Any map
    is right, also one that swaps; rows that stay are not touched.  A row
    outside its group is left and flagged (device_error_flags)."""
    tensors = list(tensors)
    index = _device_index(rows)
    if rows.dim() != 1:
        raise ValueError(f"reorder_rows: rows must be [R], got {tuple(rows.shape)}")
    R = rows.numel()
    group = max(R, 1) if group is None else group
    if not 1 <= group <= 1024 or R % group:
        raise ValueError(f"reorder_rows: {R} rows in groups of {group} (1 to 1024)")
    _refuse_out("reorder_rows", *tensors)
    if rows.dtype != torch.int32:
        rows = _indexes(rows, "rows")
    rows = rows.contiguous()
    spec = []
    for t in tensors:                                   # dozens of them, so no more than needed for each
        if t.get_device() != index:
            _device_index(rows, t)                      # says what is wrong
        shape = t.shape
        if not shape or shape[0] != R:
            raise ValueError(f"reorder_rows: every tensor must have {R} rows, got {tuple(shape)}")
        if t.is_contiguous():
            row = apart = t.nbytes // R if R else 0
        else:
            if R and not t[0].is_contiguous() or R > 1 and t.stride(0) < t[0].numel():
                raise ValueError("reorder_rows: the rows of a tensor must lie in one piece each, without overlap")
            row, apart = (t[0].nbytes if R else 0), t.stride(0) * t.element_size()
        spec += (t.data_ptr(), row, apart)
    if not spec:
        return
    if len(set(spec[::3])) < len(tensors) and len({p for p, row in zip(spec[::3], spec[1::3]) if row}) < sum(1 for row in spec[1::3] if row):
        raise ValueError("reorder_rows: a tensor is given twice")
    if rows.data_ptr() in spec[::3]:                    # the map is among what moves: the kernel reads one that does not
        rows = rows.clone()
    words = struct.pack(f"={len(spec)}q", *spec)
    _launch(index, "nt_reorder_rows", len(tensors), _bytes_address(words), R, group, rows.data_ptr())
    increment_version(tensors)


def _bytes_address(b: bytes) -> int:
    return ctypes.cast(b, ctypes.c_void_p).value


@functools.lru_cache(maxsize=256)
def _kv_fork_bytes(*sizes: int) -> int:
    return load().nt_kv_fork_workspace_bytes(*sizes)


def kv_fork(table: Tensor, refs: Tensor, lengths: Tensor, parents: Tensor, page: int, tokens: int = 1,
            window: Optional[int] = None, group: Optional[int] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """Lets row r of a cache go on from row parents[r] without copying it -> (copies [R, 2], shared [R / group]).

    In place: table int32 [R, blocks] (-1: no page), refs int32 [pages] (how many table
    entries, and other holders, have a page; 0: free) and lengths int32 [R], R at
    most 1024.  A row takes its parent's length and pages (-1: the row ends), with a
    window only those that a next token can see; pages without refs are free again.  A last
    page that is not full is made the row's own, since the next token is written there:
    one of the rows that have it keeps it when nothing else does (one that goes on from
    itself before others), the others get a new one and a line (from, to) in `copies` for
    kv_copy_pages; other lines are -1.  The next `tokens` tokens get pages (with a window
    those that it still sees behind them).  New pages are the free ones of lowest index, row
    by row.  shared: with `group`, how many leading tokens the rows of each group have in
    the same pages, for kv_attention_shared; a row that ends has none, so its group shares nothing
    (a row of no more use may go on from another of its group instead, with no new tokens).  Without enough pages or blocks entries stay -1, which is
    flagged (device_error_flags) like bad parents, lengths and pages."""
    index = _device_index(table, refs, lengths, parents)
    if table.dim() != 2 or table.dtype != torch.int32 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"kv_fork: table must be int32 [R, blocks] with unit stride, got {table.dtype} {tuple(table.shape)}")
    R, blocks = table.shape
    if R > 1024 or (R > 1 and table.stride(0) < blocks):
        raise ValueError(f"kv_fork: a table of at most 1024 rows that do not overlap, got {R}")
    if lengths.shape != (R,) or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        raise ValueError(f"kv_fork: lengths must be contiguous int32 [{R}]")
    if refs.dim() != 1 or refs.dtype != torch.int32 or not refs.is_contiguous():
        raise ValueError("kv_fork: refs must be contiguous int32 [pages]")
    if page < 1 or tokens < 0 or (window is not None and window < 0):
        raise ValueError(f"kv_fork: page {page}, tokens {tokens}, window {window}")
    if group is not None and (group < 1 or R % group):
        raise ValueError(f"kv_fork: {R} rows in groups of {group}")
    parents = _row_ints("kv_fork", "parents", _indexes(parents, "parents"), R)
    copies = torch.empty((R, 2), dtype=torch.int32, device=table.device)
    shared = ws = None
    nbytes = 0
    if group is not None:
        nbytes = _kv_fork_bytes(R, blocks, group)
        shared = torch.empty(R // group, dtype=torch.int32, device=table.device)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=table.device)
    _launch(index, "nt_kv_fork", R, refs.numel(), blocks, page, tokens, -1 if window is None else min(int(window), 2 ** 31),
            group or 0, table.data_ptr(), max(table.stride(0), blocks), refs.data_ptr(), lengths.data_ptr(), parents.data_ptr(),
            copies.data_ptr(), _ptr(shared), _ptr(ws), nbytes)
    increment_version((table, refs, lengths))
    return copies, shared


def kv_copy_pages(layers: Sequence[Tuple[Tensor, Tensor, Tensor, Tensor]], pages: Tensor) -> None:
    """Copies pages within the pools of every layer: codes and scales of keys and values.

    layers: (k_codes, k_scale, v_codes, v_scale) each, as kv_append has them and all of one shape;
    pages: int32 [N, 2], from and to, (-1, -1) is skipped (kv_fork's copies).  No page may be
    written twice, or both read and written; one outside the pool is skipped and flagged."""
    layers = list(layers)
    flat = [t for layer in layers for t in layer]
    index = _device_index(pages, *flat)
    if pages.dim() != 2 or pages.shape[1] != 2 or pages.dtype != torch.int32:
        raise ValueError(f"kv_copy_pages: pages must be int32 [N, 2], got {pages.dtype} {tuple(pages.shape)}")
    if not layers:
        return
    shape = layers[0][0].shape
    if len(shape) != 4 or shape[1] < 1 or shape[3] not in (64, 128) or shape[2] not in (16, 32, 64):
        raise ValueError(f"kv_copy_pages: codes must be [pages, heads, page of 16, 32 or 64, 64 or 128], got {tuple(shape)}")
    per_head, f8, u8, f32 = shape[:2], torch.float8_e4m3fn, torch.uint8, torch.float32
    for kc, ks, vc, vs in layers:
        for c in (kc, vc):
            dtype = c.dtype
            if c.shape != shape or dtype != f8 and dtype != u8 or not c.is_contiguous():
                raise ValueError(f"kv_copy_pages: codes must be contiguous float8_e4m3fn or uint8 {tuple(shape)}")
        for x in (ks, vs):
            if x.shape != per_head or x.dtype != f32 or not x.is_contiguous():
                raise ValueError(f"kv_copy_pages: scales must be contiguous float32 {tuple(per_head)}")
    _refuse_out("kv_copy_pages", *flat)
    spec = [t.data_ptr() for t in flat]
    if shape[0] == 0 or pages.shape[0] == 0:
        return
    pages = pages.contiguous()
    words = struct.pack(f"={len(spec)}q", *spec)
    _launch(index, "nt_kv_copy_pages", len(layers), _bytes_address(words), shape[0], shape[1], shape[2], shape[3], pages.shape[0],
            pages.data_ptr())
    increment_version(flat)


@functools.lru_cache(maxsize=256)
def _kv_attention_shared_bytes(*sizes: int) -> int:
    return load().nt_kv_attention_shared_workspace_bytes(*sizes)


def kv_attention_shared(q: Tensor, k_codes: Tensor, k_scale: Tensor, v_codes: Tensor, v_scale: Tensor, table: Tensor,
                        lengths: Tensor, shared: Tensor, counts: Optional[Tensor] = None, window: Optional[int] = None,
                        scale: Optional[float] = None) -> Tensor:
    """kv_attention for sequences that share their beginnings, which are read once -> [B, T, Hq, D].

    shared: int32 [groups], groups of B / groups consecutive sequences each (the beams of a
    prompt, say): the first shared[g] positions of a group's sequences hold the same keys and
    values, by each one's own table (kv_fork's `shared`; 0 where nothing is).  Arguments and
    results otherwise as kv_attention."""
    _refuse_grad("kv_attention_shared", q, k_codes, k_scale, v_codes, v_scale)
    index = _device_index(q, k_codes, k_scale, v_codes, v_scale, table, lengths, shared, counts)
    code = _dtype_code(q)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, T, H, D], got {tuple(q.shape)}")
    B, T, Hq, D = q.shape
    H, P, n, blocks, lengths, counts = _cache_args("kv_attention_shared", B, D, k_codes, k_scale, v_codes, v_scale, table,
                                                   lengths, counts)
    if H < 1 or Hq < H or Hq % H:
        raise ValueError(f"kv_attention_shared: {Hq} query heads over {H} cached heads")
    if window is not None and window < 0:
        raise ValueError(f"kv_attention_shared: window must be None or >= 0, got {window}")
    groups = shared.numel()
    if shared.dim() != 1 or groups < 1 or B % groups:
        raise ValueError(f"kv_attention_shared: {B} sequences do not make the groups of shared {tuple(shared.shape)}")
    shared = _indexes(shared, "shared").contiguous()
    win = -1 if window is None else min(int(window), 2 ** 31)      # as good as none from there on
    if q.stride(3) != 1:
        q = q.contiguous()
    q_sb, q_st, q_sh, _ = q.stride()
    out = _like(q)
    nbytes = _kv_attention_shared_bytes(code, B, groups, T, Hq, H, D, P, blocks, win)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(index, "nt_kv_attention_shared", code, B, groups, T, Hq, H, D, P, n, blocks, win, D ** -0.5 if scale is None else scale,
            q.data_ptr(), q_sb, q_st, q_sh, k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(),
            table.data_ptr(), table.stride(0), lengths.data_ptr(), _ptr(counts), shared.data_ptr(), out.data_ptr(), _ptr(ws), nbytes)
    return out


def launch_count() -> int:
    """Kernels this library has launched in this process (nt_launch_count)."""
    return int(load().nt_launch_count())


def bounded_wait_check(limit_ns: int, device: Optional[torch.device] = None) -> None:
    """Launch the bounded-wait check on the current stream (nt_bounded_wait_check)."""
    dev = device or torch.device("cuda", torch.cuda.current_device())
    _check("nt_bounded_wait_check", load().nt_bounded_wait_check(int(limit_ns), _stream(dev)))


def device_error_flags(device: int = 0, clear: bool = True) -> int:
    """Read the device error word set by kernels whose bounded waits expired (synchronises)."""
    v = ctypes.c_uint(0)
    _check("nt_get_error_flag", load().nt_get_error_flag(device, ctypes.byref(v), 1 if clear else 0))
    return int(v.value)
