"""Per-op entry points over torch device tensors (tests, benchmarks).

Each function is a thin call into the C ABI of libqw35cuda.so
(include/qw35_cuda.h): torch only provides the device memory and the current
stream.  There is no torch or CPU implementation behind any of them.
"""
from __future__ import annotations

import ctypes as C
import functools
import threading

import torch

from ._lib import call, check, err_buf, lib

GF4, Q8_0, Q4_K, Q5_K, Q6_K = 100, 8, 12, 13, 14
EXACT = 1


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dev(t):
    assert t.is_cuda, "device tensor expected"
    assert t.is_contiguous()
    return t


def weight_bytes(type_id: int, rows: int, k: int) -> int:
    """GGUF-layout bytes of a rows x k matrix."""
    return int(lib().qw35_cuda_weight_bytes(type_id, rows, k))


def device_bytes(type_id: int, rows: int, k: int) -> int:
    """Device-layout bytes (Q8_0 adds a per-row exponent plane)."""
    return int(lib().qw35_cuda_device_bytes(type_id, rows, k))


def repack(type_id: int, raw: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """GGUF-layout bytes (device uint8) -> device layout."""
    out = torch.empty(device_bytes(type_id, rows, k), dtype=torch.uint8, device=raw.device)
    call("qw35_cuda_weight_repack", type_id, _p(_dev(raw)), _p(out), rows, k, _stream())
    return out


def upload(type_id: int, raw_host, rows: int, k: int, device="cuda") -> torch.Tensor:
    """numpy GGUF bytes -> repacked device weight."""
    raw = torch.from_numpy(raw_host).to(device)
    return repack(type_id, raw, rows, k)


def dequant(type_id: int, w: torch.Tensor, rows: int, k: int, exact: bool = False) -> torch.Tensor:
    out = torch.empty((rows, k), dtype=torch.float32, device=w.device)
    call("qw35_cuda_dequant", type_id, _p(_dev(w)), _p(out), rows, k, EXACT if exact else 0, _stream())
    return out


def _xdtype(x):
    if x.dtype == torch.float32:
        return 0
    if x.dtype == torch.float16:
        return 1
    raise TypeError("x must be float32 or float16")


def matvec(type_id: int, w, x, rows: int, k: int, y=None, accumulate=False, exact=False):
    b = x.shape[0] if x.dim() == 2 else 1
    if y is None:
        y = torch.zeros((b, rows), dtype=torch.float32, device=x.device)
    call("qw35_cuda_matvec", type_id, _p(_dev(w)), _p(_dev(x)), _xdtype(x), _p(_dev(y)), rows, k, b,
         1 if accumulate else 0, EXACT if exact else 0, _stream())
    return y


def gate_up_swiglu(type_id: int, wg, wu, x, rows: int, k: int, exact=False):
    b = x.shape[0] if x.dim() == 2 else 1
    h = torch.empty((b, rows), dtype=torch.float32, device=x.device)
    call("qw35_cuda_gate_up_swiglu", type_id, _p(_dev(wg)), _p(_dev(wu)), _p(_dev(x)), _xdtype(x), _p(h), rows, k, b,
         EXACT if exact else 0, _stream())
    return h


def argmax_workspace(rows: int, batch: int, device="cuda"):
    n = int(lib().qw35_cuda_argmax_workspace_bytes(rows, batch))
    return torch.empty(n, dtype=torch.uint8, device=device)


def argmax_head(type_id: int, w, x, rows: int, k: int, want_logits=False, exact=False, ws=None):
    b = x.shape[0] if x.dim() == 2 else 1
    tok = torch.empty(b, dtype=torch.int32, device=x.device)
    val = torch.empty(b, dtype=torch.float32, device=x.device)
    logits = torch.empty((b, rows), dtype=torch.float32, device=x.device) if want_logits else None
    if ws is None:
        ws = argmax_workspace(rows, b, x.device)
    call("qw35_cuda_argmax_head", type_id, _p(_dev(w)), _p(_dev(x)), _p(logits), rows, k, b, _p(tok), _p(val),
         _p(ws), ws.numel(), EXACT if exact else 0, _stream())
    return tok, val, logits


def deltanet_step(proj, conv_w, dt, a, norm_w, conv_state, ssm_state, slots=None, eps=1e-6):
    """proj [n, >=12352]; conv_state [slots, 8192*3]; ssm_state [slots, 32*128*128]."""
    n = proj.shape[0]
    out = torch.empty((n, 4096), dtype=torch.float32, device=proj.device)
    call("qw35_cuda_deltanet_step", n, _p(_dev(proj)), proj.shape[1], _p(_dev(conv_w)), _p(_dev(dt)), _p(_dev(a)),
         _p(_dev(norm_w)), _p(_dev(conv_state)), conv_state[0].numel(), _p(_dev(ssm_state)), ssm_state[0].numel(),
         _p(slots), _p(out), float(eps), _stream())
    return out


def deltanet_core(q, k, v, beta, g, state):
    n = q.shape[0]
    y = torch.empty((n, 32, 128), dtype=torch.float32, device=q.device)
    call("qw35_cuda_deltanet_core", n, _p(_dev(q)), _p(_dev(k)), _p(_dev(v)), _p(_dev(beta)), _p(_dev(g)),
         _p(_dev(state)), _p(y), _stream())
    return y


def attn_preprocess(qkv, q_norm_w, k_norm_w, rope_freq, pos, chunk_ptrs, k_off, v_off, eps=1e-6, kv_q8=False):
    """kv_q8: the planes hold q8_0 rows (272 bytes per head-row) instead of f16."""
    n = qkv.shape[0]
    q = torch.empty((n, 16, 256), dtype=torch.float32, device=qkv.device)
    gate = torch.empty_like(q)
    call("qw35_cuda_attn_preprocess_q8_0" if kv_q8 else "qw35_cuda_attn_preprocess", n, _p(_dev(qkv)), qkv.shape[1], _p(_dev(q_norm_w)), _p(_dev(k_norm_w)),
         _p(_dev(rope_freq)), _p(_dev(pos)), _p(_dev(chunk_ptrs)), chunk_ptrs.shape[1], k_off, v_off, _p(q), _p(gate),
         float(eps), _stream())
    return q, gate


def gqa_workspace(n: int, max_len: int, device="cuda"):
    return torch.empty(int(lib().qw35_cuda_gqa_workspace_bytes(n, max_len)), dtype=torch.uint8, device=device)


def gqa_decode(q, gate, seq_len, max_len, chunk_ptrs, k_off, v_off, window=0, sink=0, ws=None, out=None,
               kv_q8=False):
    n = q.shape[0]
    if out is None:
        out = torch.empty((n, 4096), dtype=torch.float32, device=q.device)
    if ws is None:
        ws = gqa_workspace(n, max_len, q.device)
    call("qw35_cuda_gqa_decode_q8_0" if kv_q8 else "qw35_cuda_gqa_decode", n, _p(_dev(q)), _p(gate), _p(_dev(seq_len)), max_len, _p(_dev(chunk_ptrs)),
         chunk_ptrs.shape[1], k_off, v_off, window, sink, _p(out), _p(ws), ws.numel(), _stream())
    return out


# The calls below check their tensors on every call, so each check is a few attribute reads and nothing more: at a
# single token the wrapper is most of what a call costs (16 us of host time, 4 us on the GPU).

def _ints(t, dev, shape):
    """A device int32 index array of the given shape."""
    if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"contiguous int32 tensor of shape {shape} on cuda:{dev} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _floats(t, dev, size):
    """A device float32 vector of the given size (norm weights, frequencies)."""
    if t.dtype is not torch.float32 or t.numel() != size or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"contiguous float32 tensor of {size} values on cuda:{dev} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(t, dev):
    """A device chunk table [rows, chunks] of 64-bit addresses."""
    if t.dtype not in (torch.int64, torch.uint64) or t.dim() != 2 or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"chunk_ptrs must be a contiguous 2-d tensor of 64-bit addresses on cuda:{dev}")
    return t.data_ptr()


def _heads(t, dev, n, dtype):
    """q, gate or out: [n, 16, 256] (or [n, 4096]) values of `dtype`; None passes."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n * 4096 or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"contiguous {dtype} tensor of {n} x 16 x 256 values on cuda:{dev} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _workspace(t, dev):
    """A workspace: bytes on the tensors' device."""
    if t.dtype is not torch.uint8 or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"contiguous uint8 workspace on cuda:{dev} expected, got {t.dtype} on {t.device}")
    return t.data_ptr()


def _head_dtype(dtype):
    if dtype is torch.float32:
        return 0
    if dtype is torch.float16:
        return 1
    raise TypeError("q, gate and out must be float32 or float16")


def _device_of(t):
    if not t.is_cuda:
        raise TypeError("device tensor expected")
    return t.get_device()


class _Errors(threading.local):
    def __init__(self):
        self.buf = err_buf()


_errors = _Errors()


def _on_device(dev, func, *args):
    """call() of an entry point on device `dev` and its current stream (by its raw handle: current_stream() costs 3 us)."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _on_device(dev, func, *args)
    e = _errors.buf
    if not func(*args, torch._C._cuda_getCurrentRawStream(dev), e, 1024):
        check(0, e)


@functools.lru_cache(maxsize=64)
def _int32s(values):
    return (C.c_int32 * len(values))(*values)


def attn_append(qkv, q_norm_w, k_norm_w, rope_freq, rope_pos, sections, tok_seq, tok_pos, chunk_ptrs, k_off, v_off,
                eps=1e-6, interleaved=True, dtype=torch.float32, kv_q8=False, q=None, gate=None):
    """Append token runs to the cache; returns q and gate [n, 16, 256] as `dtype` (f32 or f16).

    qkv [n, >= 10240] f32 (rows may be strided); rope_pos [axes, n] int32 rotary positions, `sections` the pairs per
    axis; tok_seq / tok_pos [n] int32: chunk-table row (negative: padding, nothing written) and cache position.
    """
    dev = _device_of(qkv)
    shape = qkv.shape
    if qkv.dtype is not torch.float32 or len(shape) != 2 or shape[1] < 10240 or qkv.stride(1) != 1 or qkv.stride(0) >= 1 << 32:
        raise TypeError("qkv must be a float32 device tensor [n, >= 10240] with contiguous rows less than 2^32 values apart")
    n, axes, half = shape[0], len(sections), _head_dtype(dtype)
    if q is None:
        q = qkv.new_empty((n, 16, 256), dtype=dtype)
        q_ptr = q.data_ptr()
    else:
        q_ptr = _heads(q, dev, n, dtype)
    if gate is None:
        gate = torch.empty_like(q)
        gate_ptr = gate.data_ptr()
    else:
        gate_ptr = _heads(gate, dev, n, dtype)
    table = chunk_ptrs.shape
    _on_device(dev, lib().qw35_cuda_attn_append, n, qkv.data_ptr(), qkv.stride(0) if n > 1 else shape[1],
               _floats(q_norm_w, dev, 256), _floats(k_norm_w, dev, 256), _floats(rope_freq, dev, 32),
               _ints(rope_pos, dev, (axes, n)), axes, _int32s(tuple(sections)), 1 if interleaved else 0,
               _ints(tok_seq, dev, (n,)), _ints(tok_pos, dev, (n,)), table[0], _table(chunk_ptrs, dev), table[1], k_off,
               v_off, 1 if kv_q8 else 0, q_ptr, gate_ptr, half, eps)
    return q, gate


def gqa_prefill_workspace(n_row: int, n_run: int, max_run: int, max_len: int, device="cuda"):
    n = int(lib().qw35_cuda_gqa_prefill_workspace_bytes(n_row, n_run, min(max_run, n_row), max_len))
    return torch.empty(n, dtype=torch.uint8, device=device)


def gqa_prefill(q, gate, run_off, seq_len, max_run, max_len, chunk_ptrs, k_off, v_off, window=0, sink=0, ws=None,
                out=None, kv_q8=False):
    """Causal attention of token runs over the cache that already holds them; [n, 4096] in q's type.

    run_off [runs + 1], seq_len [runs] int32: rows run_off[i]..run_off[i+1] of q are the last tokens of sequence i.
    max_run, max_len: upper bounds of the runs' rows and of seq_len, max_len within the table's 256 positions a chunk.
    """
    dev, dtype = _device_of(q), q.dtype
    n, runs, table = q.shape[0], seq_len.numel(), chunk_ptrs.shape
    max_run = min(max_run, n)  # (the entry point refuses bounds that cannot be reached)
    if table[0] < runs:
        raise ValueError("chunk_ptrs needs a row for every run")
    half, L = _head_dtype(dtype), lib()
    if out is None:
        out = q.new_empty((n, 4096))
        out_ptr = out.data_ptr()
    else:
        out_ptr = _heads(out, dev, n, dtype)
    if ws is None:
        ws = q.new_empty(L.qw35_cuda_gqa_prefill_workspace_bytes(n, runs, max_run, max_len), dtype=torch.uint8)
    _on_device(dev, L.qw35_cuda_gqa_prefill, n, _heads(q, dev, n, dtype), _heads(gate, dev, n, dtype), half, runs,
               _ints(run_off, dev, (runs + 1,)), _ints(seq_len, dev, (runs,)), max_run, max_len, _table(chunk_ptrs, dev),
               table[1], k_off, v_off, 1 if kv_q8 else 0, window, sink, out_ptr, _workspace(ws, dev), ws.numel())
    return out


def gqa_decode_shared_workspace(n_seq: int, n_group: int, max_shared: int, max_own: int, device="cuda"):
    n = int(lib().qw35_cuda_gqa_decode_shared_workspace_bytes(n_seq, n_group, max_shared, max_own))
    return torch.empty(n, dtype=torch.uint8, device=device)


def gqa_decode_shared(q, gate, seq_len, group_off, shared_len, max_shared, max_own, chunk_ptrs, k_off, v_off, window=0,
                      sink=0, ws=None, out=None, kv_q8=False):
    """gqa_decode for sequences that share prefixes, each read once for 32 sequences of a group; [n, 4096] in q's type.

    group_off [groups + 1], shared_len [groups] int32: sequences group_off[g]..group_off[g+1] agree on their first
    shared_len[g] positions, all of which the first one's table row holds.  max_shared, max_own: upper bounds of
    shared_len and of seq_len - shared_len.
    """
    dev, dtype = _device_of(q), q.dtype
    n, groups, table = q.shape[0], shared_len.numel(), chunk_ptrs.shape
    if table[0] < n:
        raise ValueError("chunk_ptrs needs a row for every sequence")
    half, L = _head_dtype(dtype), lib()
    if out is None:
        out = q.new_empty((n, 4096))
        out_ptr = out.data_ptr()
    else:
        out_ptr = _heads(out, dev, n, dtype)
    if ws is None:
        ws = q.new_empty(L.qw35_cuda_gqa_decode_shared_workspace_bytes(n, groups, max_shared, max_own), dtype=torch.uint8)
    _on_device(dev, L.qw35_cuda_gqa_decode_shared, n, _heads(q, dev, n, dtype), _heads(gate, dev, n, dtype), half,
               _ints(seq_len, dev, (n,)), groups, _ints(group_off, dev, (groups + 1,)), _ints(shared_len, dev, (groups,)),
               max_shared, max_own, _table(chunk_ptrs, dev), table[1], k_off, v_off, 1 if kv_q8 else 0, window, sink,
               out_ptr, _workspace(ws, dev), ws.numel())
    return out
