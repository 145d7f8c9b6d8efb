"""Typed torch front end of the C ABI: one function per extern "C" entry point.

Each function takes CUDA tensors, checks dtypes/shapes the way the reference
does, allocates outputs on the input's device through torch's caching
allocator, and enqueues the kernel on the current stream.  The reference-named
drop-ins (FlatGate, _proto_pool_seq, direct_index_sparse_triton, ...) are thin
layers over these.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib

BLOCK = 64


def _dt(t: torch.Tensor) -> int:
    try:
        return _lib.DTYPE_CODE[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}; expected float32, bfloat16 or float16") from None


def _vec_ok(t: torch.Tensor) -> torch.Tensor:
    """A view the 16-byte vector kernels accept (copy only if it is not)."""
    es = t.element_size()
    vn = 16 // es
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % vn == 0 for s in t.stride()[:-1]):
        return t
    return t.contiguous()


def group_avg_tokens(x: torch.Tensor, G: int) -> torch.Tensor:
    """[b, H, L, d] -> [b, G, L, d] (teacher/chunked_extract.py:75-80)."""
    _lib.require_cuda(x)
    b, H, T, d = x.shape
    if H % G:
        raise AssertionError(f"H={H} not divisible by G={G}")
    x = _vec_ok(x)
    out = torch.empty((b, G, T, d), device=x.device, dtype=x.dtype)
    L = _lib.load()
    _lib.check(L.spruce_group_avg_tokens(x.data_ptr(), _lib.strides(x), _dt(x), b, H, T, d, G, out.data_ptr(),
                                         _lib.stream_of(x)))
    return out


def proto_pool(x: torch.Tensor, block: int = BLOCK, P: int = 1) -> torch.Tensor:
    """[b, H, L, d] -> [b, H, nb, P, d] (teacher/chunked_extract.py:27-72)."""
    _lib.require_cuda(x)
    b, H, T, d = x.shape
    nb = (T + block - 1) // block
    x = _vec_ok(x)
    out = torch.empty((b, H, nb, P, d), device=x.device, dtype=x.dtype)
    L = _lib.load()
    _lib.check(L.spruce_proto_pool(x.data_ptr(), _lib.strides(x), _dt(x), b, H, T, d, block, P, out.data_ptr(),
                                   _lib.stream_of(x)))
    return out


def pool_qk(q: torch.Tensor, k: torch.Tensor, P: int = 1):
    """Selector inputs: (pooled_q, pooled_k), each [B, Hkv, qb, d] (P = 1) or
    [B, Hkv, qb, P, d] (P prototypes: the mean and the P-1 farthest rows)."""
    _lib.require_cuda(q, k)
    B, Hq, T, d = q.shape
    Hkv = k.shape[1]
    if q.dtype != k.dtype:
        raise ValueError("q and k must share a dtype")
    q, k = _vec_ok(q), _vec_ok(k)
    qb = (T + BLOCK - 1) // BLOCK
    shape = (B, Hkv, qb, d) if P == 1 else (B, Hkv, qb, P, d)
    pq = torch.empty(shape, device=q.device, dtype=q.dtype)
    pk = torch.empty(shape, device=q.device, dtype=q.dtype)
    L = _lib.load()
    if P == 1:
        _lib.check(L.spruce_pool_qk(q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), _dt(q), B, Hq, Hkv,
                                    T, d, pq.data_ptr(), pk.data_ptr(), _lib.stream_of(q)))
    else:
        _lib.check(L.spruce_pool_qk_protos(q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), _dt(q), B,
                                           Hq, Hkv, T, d, P, pq.data_ptr(), pk.data_ptr(), _lib.stream_of(q)))
    return pq, pk


def gate_project(x: torch.Tensor, W: torch.Tensor) -> torch.Tensor:
    """fp32(x[..., d]) @ W[d, p] with a fixed fma order -> fp32 [..., p]."""
    _lib.require_cuda(x, W)
    d, p = W.shape
    if x.shape[-1] != d:
        raise ValueError(f"feature dim {x.shape[-1]} does not match projection {tuple(W.shape)}")
    xc = x.contiguous()
    Wc = W.detach().float().contiguous()
    out = torch.empty((*x.shape[:-1], p), device=x.device, dtype=torch.float32)
    N = xc.numel() // d if d else 0
    L = _lib.load()
    _lib.check(L.spruce_gate_project(xc.data_ptr(), _dt(xc), N, d, Wc.data_ptr(), p, out.data_ptr(),
                                     _lib.stream_of(x)))
    return out


def gate_maxsim(qp: torch.Tensor, kp: torch.Tensor, ids: torch.Tensor | None = None) -> torch.Tensor:
    """MaxSim scores: qp [R, nq, P, p], kp [R, nk, P, p] fp32 -> [R, nq, nk] (every key)
    or, with int64 candidate ids [R, nq, C], [R, nq, C] (selector/gate.py:29-101, :132-171)."""
    _lib.require_cuda(qp, kp)
    if qp.dtype != torch.float32 or kp.dtype != torch.float32:
        raise ValueError("MaxSim takes fp32 projections")
    R, nq, P, p = qp.shape
    if kp.dim() != 4 or kp.shape[0] != R or kp.shape[2:] != (P, p):
        raise ValueError(f"kp must be [{R}, nk, {P}, {p}], got {tuple(kp.shape)}")
    nk = kp.shape[1]
    qp, kp = qp.contiguous(), kp.contiguous()
    if ids is not None:
        _lib.require_cuda(ids)
        if ids.dim() != 3 or tuple(ids.shape[:2]) != (R, nq):
            raise ValueError(f"ids must be [{R}, {nq}, C], got {tuple(ids.shape)}")
        ids = ids.to(torch.int64).contiguous()
    ncols = nk if ids is None else ids.shape[2]
    out = torch.empty((R, nq, ncols), device=qp.device, dtype=torch.float32)
    _lib.check(_lib.load().spruce_gate_maxsim(qp.data_ptr(), kp.data_ptr(), None if ids is None else ids.data_ptr(),
                                              R, nq, nk, ncols, P, p, out.data_ptr(), _lib.stream_of(qp)))
    return out


def gate_scores(qp: torch.Tensor, kp: torch.Tensor) -> torch.Tensor:
    """qp [R, qb, p], kp [R, kb, p] fp32 -> [R, qb, kb] = qp.kp / sqrt(p)."""
    _lib.require_cuda(qp, kp)
    R, qb, p = qp.shape
    kb = kp.shape[1]
    qp = qp.float().contiguous()
    kp = kp.float().contiguous()
    out = torch.empty((R, qb, kb), device=qp.device, dtype=torch.float32)
    L = _lib.load()
    _lib.check(L.spruce_gate_scores(qp.data_ptr(), kp.data_ptr(), R, qb, kb, p, out.data_ptr(), _lib.stream_of(qp)))
    return out


def gate_select(qp: torch.Tensor, kp: torch.Tensor, k_selected: int, local_window: int = 0, sink_blocks: int = 1,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """qp/kp [B, G, qb, p] fp32 -> selected rows int32 [B, G, qb, K] (or into `out`)."""
    _lib.require_cuda(qp, kp)
    B, G, qb, p = qp.shape
    qp = qp.float().contiguous()
    kp = kp.float().contiguous()
    if out is None:
        out = torch.empty((B, G, qb, k_selected), device=qp.device, dtype=torch.int32)
    _check_rows_out(out, B, G, qb, k_selected)
    L = _lib.load()
    _lib.check(L.spruce_gate_select(qp.data_ptr(), kp.data_ptr(), B, G, qb, p, k_selected, local_window, sink_blocks,
                                    out.data_ptr(), _lib.int64s(*out.stride()[:3]), _lib.stream_of(qp)))
    return out


def _check_rows_out(out: torch.Tensor, B: int, G: int, qb: int, K: int) -> None:
    if out.dtype != torch.int32 or tuple(out.shape) != (B, G, qb, K) or out.stride(-1) != 1:
        raise ValueError(f"selected rows must be int32 [{B}, {G}, {qb}, {K}] with a unit last stride")


def select_workspace_bytes(q: torch.Tensor, k: torch.Tensor, proj_dim: int) -> int:
    B, _, T, d = q.shape
    need = int(_lib.load().spruce_select_workspace_bytes(B, k.shape[1], T, d, proj_dim, _dt(q)))
    if need < 0:
        raise ValueError(f"bad selector shape: q {tuple(q.shape)}, k {tuple(k.shape)}, proj_dim {proj_dim}")
    return need


def select_blocks(q: torch.Tensor, k: torch.Tensor, Wq: torch.Tensor, Wk: torch.Tensor, k_selected: int,
                  local_window: int = 0, sink_blocks: int = 1, out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None, q_blocks: tuple[int, int] | None = None) -> torch.Tensor:
    """Whole flat selector of one layer: int32 rows [B, Hkv, qb, K] (or into `out`).

    With ``q_blocks=(i0, i1)`` only rows i0..i1-1 are selected (and only the
    blocks they read are pooled and projected).
    """
    _lib.require_cuda(q, k, Wq, Wk)
    B, Hq, T, d = q.shape
    Hkv = k.shape[1]
    p = Wq.shape[1]
    if q.dtype != k.dtype:
        raise ValueError("q and k must share a dtype")
    if tuple(Wq.shape) != (d, p) or tuple(Wk.shape) != (d, p):
        raise ValueError(f"gate weights must be [{d}, p]")
    q, k = _vec_ok(q), _vec_ok(k)
    Wq = Wq.detach().float().contiguous()
    Wk = Wk.detach().float().contiguous()
    qb = (T + BLOCK - 1) // BLOCK
    if out is None:
        out = torch.empty((B, Hkv, qb, k_selected), device=q.device, dtype=torch.int32)
    _check_rows_out(out, B, Hkv, qb, k_selected)
    need = select_workspace_bytes(q, k, p)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 16), device=q.device, dtype=torch.uint8)
    i0, i1 = (0, qb) if q_blocks is None else q_blocks
    L = _lib.load()
    _lib.check(L.spruce_select_blocks_rows(q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), _dt(q), B,
                                           Hq, Hkv, T, d, Wq.data_ptr(), Wk.data_ptr(), p, k_selected, local_window,
                                           sink_blocks, out.data_ptr(), _lib.int64s(*out.stride()[:3]), i0, i1,
                                           workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                                           _lib.stream_of(q)))
    return out


def pack_selected_ids(ids: torch.Tensor, k_selected: int, local_window: int, key_blocks: int,
                      sink_blocks: int) -> torch.Tensor:
    """ids [R, qb, C] (any int dtype) -> int32 [R, qb, K] with the reference packing policy."""
    _lib.require_cuda(ids)
    R, qb, C = ids.shape
    ids64 = ids.to(torch.int64).contiguous()
    out = torch.empty((R, qb, k_selected), device=ids.device, dtype=torch.int32)
    L = _lib.load()
    _lib.check(L.spruce_pack_selected_ids(ids64.data_ptr(), R, qb, C, k_selected, local_window, key_blocks,
                                          sink_blocks, out.data_ptr(), _lib.stream_of(ids)))
    return out


def validate_first_violation(sel: torch.Tensor, local_window: int) -> tuple[int, int] | None:
    """(flat row, rule) of the first violating row of int32 [B, L, G, qb, K], or None."""
    _lib.require_cuda(sel)
    B, Ln, G, qb, K = sel.shape
    s = sel.contiguous()
    res = torch.empty(1, device=sel.device, dtype=torch.int64)
    L = _lib.load()
    _lib.check(L.spruce_validate_selected_blocks(s.data_ptr(), B, Ln, G, qb, K, local_window, res.data_ptr(),
                                                 _lib.stream_of(sel)))
    v = int(res.item())
    if v < 0:
        return None
    return v // 8, v % 8


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, indices: torch.Tensor,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None, q_blocks: tuple[int, int] | None = None,
                     peer_outs: list[int] | None = None) -> torch.Tensor:
    """Block-sparse causal GQA attention -> token-major [B, T, Hq, D].

    q [B, Hq, T, D], k/v [B, Hkv, T, D] (strided views are fine),
    indices int32 [B, Hkv, ceil(T/64), K].  With ``q_blocks=(i0, i1)`` only
    query blocks i0..i1-1 are computed (their rows of ``out``).  With
    ``peer_outs`` (device pointers of other GPUs' identically laid out output
    tensors, mapped into this process) every row is also stored there: the
    output all-gather fused into the kernel.
    """
    _lib.require_cuda(q, k, v, indices)
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = D ** -0.5
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k and v must share a dtype")
    if indices.dtype != torch.int32:
        raise ValueError("indices must be int32 [B,Hkv,ceil(T/64),K]")
    qb = (T + BLOCK - 1) // BLOCK
    if tuple(indices.shape[:3]) != (B, Hkv, qb):
        raise ValueError("indices must be int32 [B,Hkv,ceil(T/64),K]")
    if out is None:
        out = torch.empty((B, T, Hq, D), device=q.device, dtype=q.dtype)
    ostr = _lib.int64s(out.stride(0), out.stride(2), out.stride(1), out.stride(3))
    i0, i1 = (0, qb) if q_blocks is None else q_blocks
    L = _lib.load()
    if peer_outs:
        peers = (ctypes.c_void_p * len(peer_outs))(*peer_outs)
        _lib.check(L.spruce_sparse_attention_fwd_scatter(
            q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), v.data_ptr(), _lib.strides(v),
            indices.data_ptr(), _lib.strides(indices), out.data_ptr(), ostr, _dt(q), B, Hq, Hkv, T, D,
            indices.shape[-1], float(scale), i0, i1, peers, len(peer_outs),
            status.data_ptr() if status is not None else None, _lib.stream_of(q)))
        return out
    _lib.check(L.spruce_sparse_attention_fwd_rows(
        q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), v.data_ptr(), _lib.strides(v),
        indices.data_ptr(), _lib.strides(indices), out.data_ptr(), ostr, _dt(q), B, Hq, Hkv, T, D,
        indices.shape[-1], float(scale), i0, i1, status.data_ptr() if status is not None else None,
        _lib.stream_of(q)))
    return out


def residual_frontier(selected: torch.Tensor, starts: torch.Tensor, ends: torch.Tensor,
                      parents: torch.Tensor) -> torch.Tensor:
    """Maximal residual frontiers of selected_blocks rows [..., qb, K] -> int32 [..., qb, S], ID-sorted,
    -1 padded, S the largest frontier (interfaces/residual_summaries.py:122-220).  starts / ends int64
    and parents int32 [num_nodes] are the tree layout on the same device."""
    _lib.require_cuda(selected, starts, ends, parents)
    if selected.dtype != torch.int32 or selected.dim() < 2:
        raise ValueError("selected_blocks must be int32 [..., qb, K]")
    qb, K = selected.shape[-2:]
    sel = selected.contiguous()
    rows = math.prod(sel.shape[:-1])
    L = _lib.load()
    NN = starts.numel()
    stream = _lib.stream_of(sel)
    mx = torch.zeros(1, device=sel.device, dtype=torch.int32)
    _lib.check(L.spruce_residual_frontier(sel.data_ptr(), rows, K, qb, starts.data_ptr(), ends.data_ptr(),
                                          parents.data_ptr(), NN, None, 0, None, mx.data_ptr(), stream))
    S = int(mx.item())
    out = torch.empty((*sel.shape[:-1], S), device=sel.device, dtype=torch.int32)
    if S:
        _lib.check(L.spruce_residual_frontier(sel.data_ptr(), rows, K, qb, starts.data_ptr(), ends.data_ptr(),
                                              parents.data_ptr(), NN, out.data_ptr(), S, None, None, stream))
    return out


def residual_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, indices: torch.Tensor,
                              nodes: torch.Tensor, table, scale: float | None = None,
                              out: torch.Tensor | None = None, status: torch.Tensor | None = None,
                              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Block-sparse attention whose softmax also covers each row's residual summary keys
    (sparse/attention.py:164-265) -> token-major [B, T, Hq, D].

    ``nodes`` int32 [B, Hkv, qb, S] residual node ids (-1 padded); ``table`` a
    KVSummaryTable of the same K/V (keys/values fp32 [B, Hkv, nodes, P, D],
    counts/log_counts fp32 [B, nodes, P]).
    """
    _lib.require_cuda(q, k, v, indices, nodes)
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = D ** -0.5
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k and v must share a dtype")
    qb = (T + BLOCK - 1) // BLOCK
    if indices.dtype != torch.int32 or tuple(indices.shape[:3]) != (B, Hkv, qb):
        raise ValueError("indices must be int32 [B,Hkv,ceil(T/64),K]")
    if nodes.dtype != torch.int32 or nodes.dim() != 4 or tuple(nodes.shape[:3]) != (B, Hkv, qb):
        raise ValueError(f"residual nodes must be int32 [{B},{Hkv},{qb},S], got {tuple(nodes.shape)}")
    keys, values = table.keys.float().contiguous(), table.values.float().contiguous()
    counts, log_counts = table.counts.float().contiguous(), table.log_counts.float().contiguous()
    NN, P = keys.shape[2], keys.shape[3]
    if keys.shape != (B, Hkv, NN, P, D) or values.shape != keys.shape or counts.shape != (B, NN, P) \
            or log_counts.shape != counts.shape:
        raise ValueError("summary table shapes do not match q/k/v")
    _lib.require_cuda(keys, values, counts, log_counts)
    S = nodes.shape[3]
    if out is None:
        out = torch.empty((B, T, Hq, D), device=q.device, dtype=q.dtype)
    ostr = _lib.int64s(out.stride(0), out.stride(2), out.stride(1), out.stride(3))
    L = _lib.load()
    need = L.spruce_residual_workspace_bytes(B, Hkv, T, D, S, P, _dt(q))
    if need < 0:
        raise ValueError("bad residual attention shape")
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 16), device=q.device, dtype=torch.uint8)
    _lib.check(L.spruce_residual_sparse_attention_fwd(
        q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), v.data_ptr(), _lib.strides(v),
        indices.data_ptr(), _lib.strides(indices), nodes.data_ptr(), _lib.strides(nodes), S, keys.data_ptr(),
        values.data_ptr(), counts.data_ptr(), log_counts.data_ptr(), NN, P, out.data_ptr(), ostr, _dt(q), B, Hq,
        Hkv, T, D, indices.shape[-1], float(scale), workspace.data_ptr(), workspace.numel(),
        status.data_ptr() if status is not None else None, _lib.stream_of(q)))
    return out


def gate_denominator(proj_dim: int) -> float:
    return float(math.sqrt(proj_dim))


def ipc_export(t: torch.Tensor) -> tuple[bytes, int]:
    """(64-byte CUDA IPC handle of t's allocation, byte offset of t in it)."""
    _lib.require_cuda(t)
    h = ctypes.create_string_buffer(64)
    off = ctypes.c_int64(0)
    _lib.check(_lib.load().spruce_ipc_export(t.data_ptr(), h, ctypes.byref(off)))
    return h.raw, off.value


def ipc_import(handle: bytes, offset: int) -> tuple[int, int]:
    """Map a peer allocation into the current device's context: (pointer, mapping base)."""
    ptr, base = ctypes.c_void_p(), ctypes.c_void_p()
    buf = ctypes.create_string_buffer(handle, 64)
    _lib.check(_lib.load().spruce_ipc_import(buf, offset, ctypes.byref(ptr), ctypes.byref(base)))
    return ptr.value, base.value


def ipc_close(base: int) -> None:
    _lib.check(_lib.load().spruce_ipc_close(base))


def kv_summary_table(key: torch.Tensor, value: torch.Tensor, node_starts: torch.Tensor, node_ends: torch.Tensor,
                     block_size: int, prototypes: int, valid: torch.Tensor | None = None) -> dict:
    """Per-node prototype means of K and V (sparse/summaries.py:52-142).

    key/value [B, Hkv, T, D] CUDA tensors of one dtype; node_starts/node_ends
    int64 block ranges on the same device; valid bool/uint8 [B, T] or None.
    Returns the fp32 keys/values [B, Hkv, nodes, P, D], counts/log_counts
    [B, nodes, P] and int64 range_starts/range_ends [nodes, P].
    """
    _lib.require_cuda(key, value, node_starts, node_ends)
    if key.dtype != value.dtype:
        raise ValueError(f"key/value dtype mismatch: {key.dtype} vs {value.dtype}")
    B, H, T, D = key.shape
    nodes, P = node_starts.numel(), int(prototypes)
    dev = key.device
    key = key if key.stride(-1) == 1 else key.contiguous()
    value = value if value.stride(-1) == 1 else value.contiguous()
    st = node_starts.to(device=dev, dtype=torch.int64).contiguous()
    en = node_ends.to(device=dev, dtype=torch.int64).contiguous()
    vmask = None if valid is None else valid.to(device=dev, dtype=torch.uint8).contiguous()
    L = _lib.load()
    ws_bytes = int(L.spruce_kv_summary_workspace_bytes(B, H, T, D))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    out = {
        "keys": torch.empty((B, H, nodes, P, D), dtype=torch.float32, device=dev),
        "values": torch.empty((B, H, nodes, P, D), dtype=torch.float32, device=dev),
        "counts": torch.empty((B, nodes, P), dtype=torch.float32, device=dev),
        "log_counts": torch.empty((B, nodes, P), dtype=torch.float32, device=dev),
        "range_starts": torch.empty((nodes, P), dtype=torch.int64, device=dev),
        "range_ends": torch.empty((nodes, P), dtype=torch.int64, device=dev),
    }
    _lib.check(L.spruce_kv_summary_table(
        key.data_ptr(), _lib.strides(key), value.data_ptr(), _lib.strides(value),
        None if vmask is None else vmask.data_ptr(), _dt(key), B, H, T, D, block_size, P,
        st.data_ptr(), en.data_ptr(), nodes, out["keys"].data_ptr(), out["values"].data_ptr(),
        out["counts"].data_ptr(), out["log_counts"].data_ptr(), out["range_starts"].data_ptr(),
        out["range_ends"].data_ptr(), ws.data_ptr(), ws_bytes, _lib.stream_of(key)))
    return out


def tree_merge(child: torch.Tensor, radix: int = 2) -> torch.Tensor:
    """One key-tree level up (selector/tree.py:80-112): child [R, n, P, d] -> parent [R, ceil(n / radix), P, d]."""
    _lib.require_cuda(child)
    R, n, P, d = child.shape
    child = child.contiguous()
    out = torch.empty((R, (n + radix - 1) // radix, P, d), device=child.device, dtype=child.dtype)
    _lib.check(_lib.load().spruce_tree_merge(child.data_ptr(), _dt(child), R, n, P, d, radix, out.data_ptr(),
                                             _lib.stream_of(child)))
    return out


def tree_candidates(selected: torch.Tensor, radix: int, child_count: int, child_starts: torch.Tensor):
    """Children of each row's selection: (cand int64 [R, nq, S*radix], valid bool) (eval_tree_traversal.py:83-95)."""
    _lib.require_cuda(selected, child_starts)
    R, nq, S = selected.shape
    selected = selected.to(torch.int64).contiguous()
    starts = child_starts.to(device=selected.device, dtype=torch.int64).contiguous()
    cand = torch.empty((R, nq, S * radix), device=selected.device, dtype=torch.int64)
    valid = torch.empty((R, nq, S * radix), device=selected.device, dtype=torch.uint8)
    _lib.check(_lib.load().spruce_tree_candidates(selected.data_ptr(), R, nq, S, radix, child_count,
                                                  starts.data_ptr(), cand.data_ptr(), valid.data_ptr(),
                                                  _lib.stream_of(selected)))
    return cand, valid


def tree_topk(scores: torch.Tensor, valid: torch.Tensor, cand: torch.Tensor, k: int) -> torch.Tensor:
    """The level's beam: int64 [R, nq, k] candidate ids, -1 where invalid (eval_tree_traversal.py:104-108)."""
    _lib.require_cuda(scores, valid, cand)
    R, nq, C = scores.shape
    out = torch.empty((R, nq, k), device=scores.device, dtype=torch.int64)
    _lib.check(_lib.load().spruce_tree_topk(scores.contiguous().data_ptr(), valid.contiguous().data_ptr(),
                                            cand.contiguous().data_ptr(), R * nq, C, k, out.data_ptr(),
                                            _lib.stream_of(scores)))
    return out


def _on_one_device(device: int, *optional: torch.Tensor | None) -> bool:
    for t in optional:
        if t is not None and t.get_device() != device:
            return False
    return device >= 0


def _refuse_devices(*tensors: torch.Tensor | None) -> None:
    """The tensors are not on one CUDA device: say which."""
    tensors = [t for t in tensors if t is not None]
    _lib.require_cuda(*tensors)
    raise ValueError(f"tensors on {', '.join(sorted({str(t.device) for t in tensors}))}")


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _status_ptr(t: torch.Tensor | None) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.numel() < 1:
        raise ValueError("status must be an int32 tensor of at least one element")
    return t.data_ptr()


def _head_weight(w: torch.Tensor | None, D: int, name: str) -> torch.Tensor | None:
    if w is None:
        return None
    if tuple(w.shape) != (D,):
        raise ValueError(f"{name} must be [{D}], got {tuple(w.shape)}")
    if w.dtype == torch.float32 and w.is_contiguous():
        return w
    return w.detach().float().contiguous()


def _check_rope(rope: torch.Tensor, D: int) -> None:
    if rope.dim() != 2 or rope.dtype != torch.float32 or not rope.is_contiguous():
        raise ValueError("the rotation table must be contiguous float32 [positions, rotary width]")
    if rope.shape[1] > D or rope.shape[1] % 2:
        raise ValueError(f"rotary width {rope.shape[1]} must be even and at most head_dim {D}")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor, positions: torch.Tensor | None = None, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = False, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Head norms (where a weight is given) and rotary positions of q [B, Hq, T, D] and k [B, Hkv, T, D].

    ``rope`` fp32 [positions, rd] is ``rope.rope_table``'s: the first rd dims are rotated, pairs (i, i + rd/2), or
    (2i, 2i+1) when ``interleaved``.  ``positions`` int [B, T] or [T]; None: token t is at position t.  Returns
    token-major tensors viewed as [B, H, T, D] (the layout the selector and the attention take), or
    ``q_out`` / ``k_out``, which may be q and k themselves.
    """
    device = q.get_device()
    if not (device == k.get_device() == rope.get_device()
            and _on_one_device(device, positions, q_weight, k_weight, q_out, k_out, status)):
        _refuse_devices(q, k, rope, positions, q_weight, k_weight, q_out, k_out, status)
    B, Hq, T, D = q.shape
    dtype, ks = q.dtype, k.shape
    if dtype != k.dtype:
        raise ValueError("q and k must share a dtype")
    if len(ks) != 4 or ks[0] != B or ks[2] != T or ks[3] != D:
        raise ValueError(f"k must be [{B}, Hkv, {T}, {D}], got {tuple(ks)}")
    Hkv = ks[1]
    _check_rope(rope, D)
    q_weight, k_weight = _head_weight(q_weight, D, "q_weight"), _head_weight(k_weight, D, "k_weight")
    pos_strides = (0, 0)
    if positions is not None:
        if tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
        if positions.is_floating_point():
            raise ValueError("positions must be integers")
        positions = positions.to(torch.int64).expand(B, T)
        pos_strides = positions.stride()
    elif T > rope.shape[0]:
        raise ValueError(f"{T} tokens need a rotation table of as many positions, got {rope.shape[0]}")
    q = q if q.stride(3) == 1 else q.contiguous()
    k = k if k.stride(3) == 1 else k.contiguous()
    if q_out is None:
        q_out = q.new_empty_strided((B, Hq, T, D), (T * Hq * D, D, Hq * D, 1))
    elif q_out.shape != q.shape or q_out.dtype != dtype or q_out.stride(3) != 1:
        raise ValueError(f"an output must be {dtype} {tuple(q.shape)} with a unit last stride")
    if k_out is None:
        k_out = q.new_empty_strided((B, Hkv, T, D), (T * Hkv * D, D, Hkv * D, 1))
    elif k_out.shape != k.shape or k_out.dtype != dtype or k_out.stride(3) != 1:
        raise ValueError(f"an output must be {dtype} {tuple(k.shape)} with a unit last stride")
    args = _lib.QK_NORM_ROPE_ARGS.pack(
        q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), rope.data_ptr(), _ptr(positions),
        _ptr(q_weight), _ptr(k_weight), _status_ptr(status), _lib.stream_on(device), *q.stride(), *k.stride(),
        *q_out.stride(), *k_out.stride(), *pos_strides, _dt(q), B, Hq, Hkv, T, D, *rope.shape, interleaved, eps)
    _lib.launch(_lib.load().spruce_qk_norm_rope, args, device)
    return q_out, k_out


def _paged_shapes(k_cache, v_cache, block_table, cu_q, kv_lens, dtype):
    """A paged cache and its metadata, checked: its shape, both caches' strides, S and the table's (stride, width)."""
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("the caches must be [pages, Hkv, page_size, D] of one shape")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("the caches must have the new tokens' dtype")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the caches need a unit last stride")
    if not (block_table.dtype is cu_q.dtype is kv_lens.dtype is torch.int32):
        raise ValueError("block_table, cu_q and kv_lens must be int32")
    table, S = block_table.shape, kv_lens.numel()
    if len(table) != 2 or table[0] != S or cu_q.shape != (S + 1,) or kv_lens.dim() != 1:
        raise ValueError(f"expected block_table [S, pages], cu_q [S + 1] and kv_lens [S], got "
                         f"{tuple(table)}, {tuple(cu_q.shape)}, {tuple(kv_lens.shape)}")
    step, unit = block_table.stride()
    if unit != 1 and table[1] > 1 or not (cu_q.is_contiguous() and kv_lens.is_contiguous()):
        raise ValueError("block_table needs a unit last stride, cu_q and kv_lens must be contiguous")
    return shape, ks, vs, S, step, table[1]


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                 q: torch.Tensor | None = None, rope: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                 q_out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write new keys and values [N, Hkv, D] into a paged cache, normed and rotated on the way; returns q likewise.

    The packed tokens of sequence s are ``cu_q[s] .. cu_q[s+1]`` (those before ``cu_q[0]`` or past ``cu_q[-1]`` are left
    out, in the result too); ``kv_lens[s]`` is its length after the call, so its token i lands at position ``kv_lens[s] - q_len + i`` (page ``block_table[s, position // page_size]`` of
    ``k_cache`` / ``v_cache`` [pages, Hkv, page_size, D]).  ``rope`` None: no rotation.  ``positions`` int [N]
    replaces the cache positions in the rotation only.  With ``q`` [N, Hq, D], its norm and rotation run in the
    same launch into ``q_out`` (a new [N, Hq, D] tensor by default; q itself is allowed).
    """
    device = k.get_device()
    if not (device == v.get_device() == k_cache.get_device() == v_cache.get_device() == block_table.get_device()
            == cu_q.get_device() == kv_lens.get_device()
            and _on_one_device(device, q, rope, positions, q_weight, k_weight, q_out, status)):
        _refuse_devices(k, v, k_cache, v_cache, block_table, cu_q, kv_lens, q, rope, positions, q_weight, k_weight,
                        q_out, status)
    dtype, shape = k.dtype, k.shape
    (pages, Hkv, page_size, D), kc_strides, vc_strides, S, step, width = _paged_shapes(k_cache, v_cache, block_table,
                                                                                       cu_q, kv_lens, dtype)
    if len(shape) != 3 or shape[1] != Hkv or shape[2] != D or v.shape != shape or v.dtype != dtype:
        raise ValueError(f"k and v must be [N, {Hkv}, {D}] of one dtype, got {tuple(shape)} and {tuple(v.shape)}")
    N = shape[0]
    kn, kh, kd = k.stride()
    if kd != 1:
        k = k.contiguous()
        kn, kh, _ = k.stride()
    vn, vh, vd = v.stride()
    if vd != 1:
        v = v.contiguous()
        vn, vh, _ = v.stride()
    q_weight, k_weight = _head_weight(q_weight, D, "q_weight"), _head_weight(k_weight, D, "k_weight")
    table_rows = rd = Hq = 0
    if rope is not None:
        _check_rope(rope, D)
        table_rows, rd = rope.shape
    if positions is not None:
        if tuple(positions.shape) != (N,) or positions.is_floating_point():
            raise ValueError(f"positions must be integers [{N}]")
        positions = positions.to(torch.int64).contiguous()
    qn = qh = on = oh = 0
    if q is not None:
        shape = q.shape
        if len(shape) != 3 or shape[0] != N or shape[2] != D or q.dtype != dtype:
            raise ValueError(f"q must be {dtype} [{N}, Hq, {D}], got {q.dtype} {tuple(shape)}")
        Hq = shape[1]
        qn, qh, qd = q.stride()
        if qd != 1:
            q = q.contiguous()
            qn, qh, _ = q.stride()
        if q_out is None:
            q_out = q.new_empty((N, Hq, D))
            on, oh = Hq * D, D
        elif q_out.shape != shape or q_out.dtype != dtype or q_out.stride(2) != 1:
            raise ValueError(f"q_out must be {dtype} {tuple(shape)} with a unit last stride")
        else:
            on, oh, _ = q_out.stride()
    elif q_out is not None:
        raise ValueError("q_out without q")
    args = _lib.PAGED_APPEND_ARGS.pack(
        _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(q_out), k_cache.data_ptr(), v_cache.data_ptr(), _ptr(rope),
        _ptr(positions), _ptr(q_weight), _ptr(k_weight), block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(),
        _status_ptr(status), _lib.stream_on(device), qn, qh, kn, kh, vn, vh, on, oh, *kc_strides[:3],
        *vc_strides[:3], _dt(k), N, S, Hq, Hkv, D, pages, page_size, step, width, table_rows, rd, interleaved, eps)
    _lib.launch(_lib.load().spruce_paged_append, args, device)
    return q_out


@functools.lru_cache(maxsize=256)
def _paged_workspace_bytes(Hq: int, Hkv: int, D: int, max_q_len: int, dtype: int) -> int:
    return int(_lib.load().spruce_paged_attention_workspace_bytes(Hq, Hkv, D, max_q_len, dtype))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_lens: torch.Tensor, *, max_q_len: int, max_kv_len: int,
                    scale: float | None = None, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None, status: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of packed new tokens q [N, Hq, D] over a paged cache (see :func:`paged_append`).

    The last new token of sequence s sees ``kv_lens[s]`` keys, the one before it one fewer, and so on; queries that
    see none give zeros.  ``max_q_len`` and ``max_kv_len`` bound the sequences' new tokens and lengths (the lengths
    themselves stay on the device); longer ones are cut to them, their queries past ``max_q_len`` are not written, and only
    ``status`` says so.  Returns [N, Hq, D]; rows before ``cu_q[0]`` and past ``cu_q[-1]`` are not written.
    ``lse`` float32 [N, Hq] receives each row's log of the softmax sum (natural; -inf where it sees nothing), which
    :func:`paged_key_mass` takes.
    """
    device = q.get_device()
    if not (device == k_cache.get_device() == v_cache.get_device() == block_table.get_device() == cu_q.get_device()
            == kv_lens.get_device() and _on_one_device(device, out, workspace, status, lse)):
        _refuse_devices(q, k_cache, v_cache, block_table, cu_q, kv_lens, out, workspace, status, lse)
    dtype, shape = q.dtype, q.shape
    (pages, Hkv, page_size, D), kc_strides, vc_strides, S, step, width = _paged_shapes(k_cache, v_cache, block_table,
                                                                                       cu_q, kv_lens, dtype)
    if len(shape) != 3 or shape[2] != D:
        raise ValueError(f"q must be [N, Hq, {D}], got {tuple(shape)}")
    N, Hq, _ = shape
    dt, size = _dt(q), q.element_size()
    qn, qh, qd = q.stride()
    if qd != 1 or (qn | qh) % (16 // size) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # contiguous() returns a q at an odd address as it is
        qn, qh, _ = q.stride()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        on, oh = Hq * D, D
    elif out.shape != shape or out.dtype != dtype or out.stride(2) != 1:
        raise ValueError(f"out must be {dtype} {tuple(shape)} with a unit last stride")
    else:
        on, oh, _ = out.stride()
    if workspace is None:
        nbytes = _paged_workspace_bytes(Hq, Hkv, D, max_q_len, dt)
        if nbytes < 0:
            raise ValueError(f"bad paged attention shape: q {tuple(shape)}, cache {tuple(k_cache.shape)}, "
                             f"max_q_len {max_q_len}")
        workspace = q.new_empty(nbytes // size)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    else:
        nbytes = workspace.nbytes
    fields = (
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), cu_q.data_ptr(),
        kv_lens.data_ptr(), workspace.data_ptr(), _status_ptr(status), _lib.stream_on(device), qn, qh, *kc_strides[:3],
        *vc_strides[:3], on, oh, dt, N, S, Hq, Hkv, D, pages, page_size, step, width, max_q_len, max_kv_len, nbytes,
        D ** -0.5 if scale is None else scale)
    if lse is None:
        _lib.launch(_lib.load().spruce_paged_attention, _lib.PAGED_ATTENTION_ARGS.pack(*fields), device)
    else:
        _check_lse(lse, N, Hq)
        _lib.launch(_lib.load().spruce_paged_attention_lse,
                    _lib.PAGED_ATTENTION_LSE_ARGS.pack(*fields, lse.data_ptr(), *lse.stride()), device)
    return out


def _check_lse(lse: torch.Tensor, N: int, Hq: int) -> None:
    if tuple(lse.shape) != (N, Hq) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 [{N}, {Hq}], got {lse.dtype} {tuple(lse.shape)}")


def _check_mass(mass: torch.Tensor, shape, name: str) -> None:
    if tuple(mass.shape) != tuple(shape[:3]) or mass.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 {tuple(shape[:3])}, got {mass.dtype} {tuple(mass.shape)}")


def paged_key_mass(q: torch.Tensor, k_cache: torch.Tensor, mass: torch.Tensor, block_table: torch.Tensor,
                   cu_q: torch.Tensor, kv_lens: torch.Tensor, lse: torch.Tensor, *, max_q_len: int, max_kv_len: int,
                   decay: float = 1.0, scale: float | None = None, out: torch.Tensor | None = None,
                   status: torch.Tensor | None = None) -> torch.Tensor:
    """Add the softmax weight that cached keys receive from the new tokens q [N, Hq, D] to ``mass`` [pages, Hkv, page_size].

    ``mass'[j] = decay * mass[j] + sum over queries i that see j and heads h of j's group of exp(scale q_ih.k_j - lse_ih)``
    for each slot of a sequence with new tokens; the new tokens' own slots start from 0.  With ``decay`` 0 nothing old
    is read.  The batch is described as for :func:`paged_attention`, whose ``lse`` [N, Hq] this takes.  ``out`` (``mass`` itself
    by default) receives the sums; slots of no such sequence are left as they are.  No page may belong to two sequences of
    the call: both would write its weights.
    """
    out = mass if out is None else out
    device = q.get_device()
    if not (device == k_cache.get_device() == mass.get_device() == block_table.get_device() == cu_q.get_device()
            == kv_lens.get_device() == lse.get_device() == out.get_device() and _on_one_device(device, status)):
        _refuse_devices(q, k_cache, mass, block_table, cu_q, kv_lens, lse, out, status)
    dtype, shape = q.dtype, q.shape
    (pages, Hkv, page_size, D), kc_strides, _, S, step, width = _paged_shapes(k_cache, k_cache, block_table, cu_q,
                                                                              kv_lens, dtype)
    if len(shape) != 3 or shape[2] != D:
        raise ValueError(f"q must be [N, Hq, {D}], got {tuple(shape)}")
    N, Hq, _ = shape
    _check_lse(lse, N, Hq)
    _check_mass(mass, k_cache.shape, "mass")
    _check_mass(out, k_cache.shape, "out")
    dt, size = _dt(q), q.element_size()
    qn, qh, qd = q.stride()
    if qd != 1 or (qn | qh) % (16 // size) or q.data_ptr() % 16 or min(qn, qh) < 1:
        q = q.clone(memory_format=torch.contiguous_format)
        qn, qh, _ = q.stride()
    args = _lib.PAGED_KEY_MASS_ARGS.pack(
        q.data_ptr(), k_cache.data_ptr(), lse.data_ptr(), mass.data_ptr(), out.data_ptr(), block_table.data_ptr(),
        cu_q.data_ptr(), kv_lens.data_ptr(), _status_ptr(status), _lib.stream_on(device), qn, qh, *kc_strides[:3],
        *lse.stride(), *mass.stride(), *out.stride(), dt, N, S, Hq, Hkv, D, pages, page_size, step, width, max_q_len,
        max_kv_len, D ** -0.5 if scale is None else scale, decay)
    _lib.launch(_lib.load().spruce_paged_key_mass, args, device)
    return out


def paged_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, mass: torch.Tensor, block_table: torch.Tensor,
                kv_lens: torch.Tensor, keep: int, *, max_kv_len: int, sinks: int = 0, recent: int = 0,
                into: tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cut sequences of a paged cache to ``keep`` tokens, each KV head to the ones of the largest ``mass``.

    A sequence longer than ``keep`` keeps its first ``sinks`` slots, its last ``recent`` ones and the heaviest of those
    between (ties: the lowest slot).  K, V and mass rows that stay move, in their order, to the first slots: in place, or
    of the pages of ``into = (k, v, mass, block_table)``, which no sequence of the call reads.  In place, no
    page may belong to two sequences.  ``kv_lens`` int32 [S] are the lengths, at most ``max_kv_len`` (a longer one is left as
    it is, and only ``status`` says so).  Returns ``kept`` int32 [S, Hkv, min(keep, max_kv_len)], the old slots (-1 past
    them), and the new lengths int32 [S].
    """
    k_out, v_out, mass_out, out_table = (k_cache, v_cache, mass, block_table) if into is None else into
    device = k_cache.get_device()
    if not (device == v_cache.get_device() == mass.get_device() == block_table.get_device() == kv_lens.get_device()
            == k_out.get_device() == v_out.get_device() == mass_out.get_device() == out_table.get_device()
            and _on_one_device(device, status)):
        _refuse_devices(k_cache, v_cache, mass, block_table, kv_lens, k_out, v_out, mass_out, out_table, status)
    shape, to_shape = k_cache.shape, k_out.shape
    if len(shape) != 4 or v_cache.shape != shape or len(to_shape) != 4 or v_out.shape != to_shape:
        raise ValueError("the caches must be [pages, Hkv, page_size, D] of one shape")
    pages, Hkv, page_size, D = shape
    if to_shape[1:] != shape[1:]:
        raise ValueError(f"the caches of `into` must be [pages, {Hkv}, {page_size}, {D}], got {tuple(to_shape)}")
    if not k_cache.dtype == v_cache.dtype == k_out.dtype == v_out.dtype:
        raise ValueError("the caches must share a dtype")
    ks, vs = k_cache.stride(), v_cache.stride()
    kos, vos = (ks, vs) if into is None else (k_out.stride(), v_out.stride())
    if not ks[3] == vs[3] == kos[3] == vos[3] == 1:
        raise ValueError("the caches need a unit last stride")
    _check_mass(mass, shape, "mass")
    _check_mass(mass_out, to_shape, "the mass of `into`")
    S = kv_lens.numel()
    for table in (block_table,) if into is None else (block_table, out_table):
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != S:
            raise ValueError(f"a block table must be int32 [{S}, pages], got {table.dtype} {tuple(table.shape)}")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("a block table needs a unit last stride")
    if kv_lens.dtype != torch.int32 or kv_lens.dim() != 1 or not kv_lens.is_contiguous():
        raise ValueError("kv_lens must be contiguous int32 [S]")
    keep, max_kv_len = int(keep), int(max_kv_len)
    if keep < 0 or max_kv_len < 0:
        raise ValueError("keep and max_kv_len must not be negative")
    kept = kv_lens.new_empty((S, Hkv, min(keep, max_kv_len)))
    lens = kv_lens.new_empty(S)
    args = _lib.PAGED_EVICT_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), mass.data_ptr(), k_out.data_ptr(), v_out.data_ptr(),
        mass_out.data_ptr(), block_table.data_ptr(), out_table.data_ptr(), kv_lens.data_ptr(), kept.data_ptr(),
        lens.data_ptr(), _status_ptr(status), _lib.stream_on(device), *ks[:3], *vs[:3],
        *mass.stride(), *kos[:3], *vos[:3], *mass_out.stride(), _dt(k_cache), S, Hkv, D, pages,
        page_size, block_table.stride(0), block_table.shape[1], to_shape[0], out_table.stride(0), out_table.shape[1],
        max_kv_len, kept.shape[2], keep, sinks, recent)
    _lib.launch(_lib.load().spruce_paged_evict, args, device)
    return kept, lens


@functools.lru_cache(maxsize=256)
def _block_mass_workspace_bytes(B: int, Hq: int, Hkv: int, T: int, D: int, dtype: int) -> int:
    return int(_lib.load().spruce_block_mass_workspace_bytes(B, Hq, Hkv, T, D, dtype))


def block_mass(q: torch.Tensor, k: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Softmax weight of whole key blocks of 64 tokens, the teacher of a gate: float32 [B, Hkv, qb, qb].

    ``out[b, g, i, j]`` is the mean over the heads of group g and the tokens of query block i of the weight that causal
    attention of q [B, Hq, T, D] over k [B, Hkv, T, D] gives to key block j; rows sum to 1.
    """
    device = q.get_device()
    if not (device == k.get_device() and _on_one_device(device, out, workspace, status)):
        _refuse_devices(q, k, out, workspace, status)
    shape, ks = q.shape, k.shape
    if len(shape) != 4 or len(ks) != 4:
        raise ValueError("q and k must be [B, H, T, D]")
    B, Hq, T, D = shape
    Hkv = ks[1]
    if q.dtype != k.dtype:
        raise ValueError("q and k must share a dtype")
    if ks[0] != B or ks[2] != T or ks[3] != D:
        raise ValueError(f"k must be [{B}, Hkv, {T}, {D}], got {tuple(ks)}")
    dt, qb = _dt(q), (T + BLOCK - 1) // BLOCK
    q, q_strides = _tma_ok(q)
    k, k_strides = _tma_ok(k)
    if out is None:
        out = q.new_empty((B, Hkv, qb, qb), dtype=torch.float32)
    elif tuple(out.shape) != (B, Hkv, qb, qb) or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError(f"out must be contiguous float32 {(B, Hkv, qb, qb)}")
    if workspace is None:
        nbytes = _block_mass_workspace_bytes(B, Hq, Hkv, T, D, dt)
        if nbytes < 0:
            raise ValueError(f"bad block mass shape: q {tuple(shape)}, k {tuple(ks)}")
        workspace = q.new_empty(nbytes // 4, dtype=torch.float32)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    else:
        nbytes = workspace.nbytes
    args = _lib.BLOCK_MASS_ARGS.pack(
        q.data_ptr(), k.data_ptr(), out.data_ptr(), workspace.data_ptr(), _status_ptr(status), _lib.stream_on(device),
        *q_strides, *k_strides, dt, B, Hq, Hkv, T, D, nbytes, D ** -0.5 if scale is None else scale)
    _lib.launch(_lib.load().spruce_block_mass, args, device)
    return out


def _tma_ok(t: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """[B, H, T, D] with 16-byte aligned rows that steps forwards (a copy only if it is not), and strides to say so."""
    vn = 16 // t.element_size()
    (b, h, n, d), (sb, sh, sn, sd) = t.shape, t.stride()
    # A dimension of one element never steps: any stride will do.
    sb, sh, sn = sb if b > 1 else d, sh if h > 1 else d, sn if n > 1 else d
    if sd == 1 and t.data_ptr() % 16 == 0 and not (sb | sh | sn) % vn and min(sb, sh, sn) > 0:
        return t, (sb, sh, sn, 1)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, (h * n * d, n * d, d, 1)


def _row_major(t: torch.Tensor, rows: int) -> torch.Tensor:
    """[..., n] as [rows, n] with a unit last stride."""
    if t.dim() != 2:
        t = t.reshape(rows, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _distill(scores, ids, teacher, visible, temperature, status, *, loss=False, stats=None, want_stats=False,
             weight=None):
    """One call of spruce_topk_distill on checked arguments: (loss, stats, grad), None where not asked for."""
    device = scores.get_device()
    if not (device == ids.get_device() == teacher.get_device()
            and _on_one_device(device, visible, stats, weight, status)):
        _refuse_devices(scores, ids, teacher, visible, stats, weight, status)
    shape, ids_shape = scores.shape, ids.shape
    lead = shape[:-1]
    if len(shape) < 1 or len(ids_shape) != len(shape) or ids_shape[:-1] != lead or teacher.shape != ids_shape:
        raise ValueError(f"expected scores [..., n], ids [..., K] and teacher [..., K], got {tuple(shape)}, "
                         f"{tuple(ids_shape)}, {tuple(teacher.shape)}")
    ids64 = ids.dtype is torch.int64
    if not ids64 and ids.dtype is not torch.int32:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    n, K = shape[-1], ids_shape[-1]
    flat = len(lead) == 1
    R = lead[0] if flat else math.prod(lead)
    if visible is not None:
        if visible.dtype is not torch.int32 or visible.shape != lead:
            raise ValueError(f"visible must be int32 {tuple(lead)}, got {visible.dtype} {tuple(visible.shape)}")
        visible = visible.contiguous() if flat else visible.reshape(R).contiguous()
    step = 0
    if weight is not None:
        if weight.dtype is not torch.float32 or weight.shape != lead:
            raise ValueError(f"the rows' weights must be float32 {tuple(lead)}, got {weight.dtype} {tuple(weight.shape)}")
        weight = weight if flat else weight.reshape(R)
        step = weight.stride(0)
    x, i, t = _row_major(scores, R), _row_major(ids, R), _row_major(teacher, R)
    out = scores.new_empty(lead, dtype=torch.float32) if loss else None
    made = scores.new_empty((R, 2), dtype=torch.float32) if want_stats else None
    grad = scores.new_empty(shape) if weight is not None else None
    args = _lib.TOPK_DISTILL_ARGS.pack(
        x.data_ptr(), i.data_ptr(), t.data_ptr(), _ptr(visible), _ptr(out), _ptr(made), _ptr(stats), _ptr(weight),
        _ptr(grad), _status_ptr(status), _lib.stream_on(device), x.stride(0), i.stride(0), t.stride(0), step, n, _dt(x), _dt(t),
        ids64, R, n, K, temperature)
    _lib.launch(_lib.load().spruce_topk_distill, args, device)
    return out, made, grad


def topk_distill(scores: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, visible: torch.Tensor | None = None,
                 temperature: float = 1.0, grad_weight: torch.Tensor | None = None,
                 status: torch.Tensor | None = None):
    """Distillation of a teacher's top entries into rows of scores [..., n]: the rows' losses float32 [...].

    With p the softmax of ``teacher`` [..., K] / temperature over the entries whose ``ids`` [..., K] are not negative, and q
    the softmax of scores / temperature over the first ``visible`` [...] columns (all by default), a row's loss is
    ``sum_k p_k (ln p_k - ln q[ids_k])``.  A column named twice counts twice; one past the visible ones counts as padding, and
    only ``status`` says so.  Rows without a visible score or a teacher entry above -inf have loss and gradient 0.

    With ``grad_weight`` float32 [...], returns ``(loss, grad)``, grad [..., n] being the gradient of the sum of
    ``grad_weight * loss`` by the scores, in the scores' dtype: both in one pass over the scores.  Not recorded by autograd;
    :func:`spruce_research_b200.selector.loss.topk_distill_loss` is.
    """
    loss, _, grad = _distill(scores, ids, teacher, visible, temperature, status, loss=True, weight=grad_weight)
    return loss if grad_weight is None else (loss, grad)


def topk_distill_forward(scores, ids, teacher, *, visible=None, temperature=1.0, status=None):
    """``(loss, stats)``: as :func:`topk_distill`, with what :func:`topk_distill_backward` needs of the scores' softmax."""
    loss, stats, _ = _distill(scores, ids, teacher, visible, temperature, status, loss=True, want_stats=True)
    return loss, stats


def topk_distill_backward(scores, ids, teacher, stats, weight, *, visible=None, temperature=1.0, status=None):
    """Gradient [..., n] of the sum of ``weight * loss`` by the scores; ``stats`` are of the forward call on them."""
    R = math.prod(scores.shape[:-1])
    if tuple(stats.shape) != (R, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats must be contiguous float32 [{R}, 2]")
    return _distill(scores, ids, teacher, visible, temperature, status, stats=stats, weight=weight)[2]
