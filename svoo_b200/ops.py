"""Torch-tensor front end of the C ABI: one function per entry point.

Tensors are CUDA, contiguous; token tensors are bf16 [BH, N, 128].  Work is enqueued
on torch's current stream; nothing here synchronises with the host.
"""
from __future__ import annotations

import ctypes
import dataclasses
import functools
from typing import Dict, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from ._lib import LIB, check

HEAD_DIM = 128
_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("svoo_b200 ops need CUDA tensors; there is no CPU path")
        if not t.is_contiguous():
            raise ValueError("svoo_b200 ops need contiguous tensors")


def _tokens(x: torch.Tensor) -> Tuple[int, int, int]:
    if x.dim() != 3 or x.dtype != torch.bfloat16:
        raise ValueError(f"expected bf16 [BH, N, {HEAD_DIM}] tokens, got {x.dtype} {tuple(x.shape)}")
    return x.shape


def rows_in_place(x: torch.Tensor) -> bool:
    """Whether the clustering can read x [BH, N, 128] where it is: CUDA, dense rows, heads a whole number
    (>= N) of rows apart -- a tensor of its own or the leading rows of longer per-head sequences."""
    return (x.is_cuda and x.dim() == 3 and x.shape[-1] == HEAD_DIM and x.stride(-1) == 1 and
            (x.shape[1] == 1 or x.stride(1) == HEAD_DIM) and x.data_ptr() % 16 == 0 and
            (x.shape[0] == 1 or (x.stride(0) % HEAD_DIM == 0 and x.stride(0) >= x.shape[1] * HEAD_DIM and
                                 x.shape[0] * x.stride(0) // HEAD_DIM < 2 ** 31 and x.stride(0) // HEAD_DIM <= 1 << 24)))


def workspace_bytes(BH: int, N: int, QC: int, KC: int) -> int:
    out = ctypes.c_int64(0)
    check(LIB.svoo_b200_workspace_bytes(BH, N, QC, KC, ctypes.byref(out)), "workspace_bytes")
    return out.value


def workspace(device: torch.device, BH: int, N: int, QC: int, KC: int) -> torch.Tensor:
    """A cached uint8 scratch tensor of at least the needed size, one per device and stream."""
    need = workspace_bytes(BH, N, QC, KC)
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


@dataclasses.dataclass
class Clustering:
    """Everything one co-clustering call produces (all on device)."""
    qlabels: torch.Tensor      # int32 [BH, N]
    klabels: torch.Tensor
    qcentroids: torch.Tensor   # bf16 [BH, QC, 128]
    kcentroids: torch.Tensor
    qsizes: torch.Tensor       # int32 [BH, QC]
    ksizes: torch.Tensor
    q_sorted_idx: torch.Tensor  # int32 [BH, N] stable cluster-order permutation
    k_sorted_idx: torch.Tensor
    q_offsets: torch.Tensor     # int32 [BH, QC+1]
    k_offsets: torch.Tensor


def cocluster(q: torch.Tensor, k: torch.Tensor, q_init_idx: Optional[torch.Tensor],
              k_init_idx: Optional[torch.Tensor], iters: int,
              init_centroids: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Clustering:
    """Co-clustering from initial centroid token indices, or (warm start) from `init_centroids` =
    (q centroids [BH,QC,128], k centroids [BH,KC,128]), which are not modified.  q and k may be the leading
    rows of longer per-head sequences (rows_in_place), spaced alike."""
    if not (rows_in_place(q) and rows_in_place(k) and (q.shape[0] == 1 or q.stride(0) == k.stride(0))):
        _need_cuda(q, k)
    BH, N, D = _tokens(q)
    if k.shape != q.shape or k.dtype != q.dtype:
        raise ValueError("q and k must have the same shape and dtype")
    head_rows = N if BH == 1 else q.stride(0) // HEAD_DIM
    dev = q.device
    i32 = dict(dtype=torch.int32, device=dev)
    if init_centroids is not None:
        qc0, kc0 = init_centroids
        _need_cuda(qc0, kc0)
        QC, KC = qc0.shape[1], kc0.shape[1]
        if qc0.shape != (BH, QC, D) or kc0.shape != (BH, KC, D) or qc0.dtype != q.dtype or kc0.dtype != q.dtype:
            raise ValueError("initial centroids must be bf16 [BH, QC, 128] and [BH, KC, 128]")
        qcent, kcent = qc0.clone(), kc0.clone()
        qi_ptr = ki_ptr = 0
    else:
        if q_init_idx is None or k_init_idx is None:
            raise ValueError("cocluster needs both initial index tensors, or init_centroids")
        _need_cuda(q_init_idx, k_init_idx)
        QC, KC = q_init_idx.shape[-1], k_init_idx.shape[-1]
        qi = q_init_idx.to(torch.int32).contiguous()
        ki = k_init_idx.to(torch.int32).contiguous()
        qi_ptr, ki_ptr = qi.data_ptr(), ki.data_ptr()
        qcent = torch.empty(BH, QC, D, dtype=q.dtype, device=dev)
        kcent = torch.empty(BH, KC, D, dtype=q.dtype, device=dev)
    c = Clustering(
        torch.empty(BH, N, **i32), torch.empty(BH, N, **i32), qcent, kcent,
        torch.empty(BH, QC, **i32), torch.empty(BH, KC, **i32),
        torch.empty(BH, N, **i32), torch.empty(BH, N, **i32),
        torch.empty(BH, QC + 1, **i32), torch.empty(BH, KC + 1, **i32))
    ws = workspace(dev, BH, N, QC, KC)
    check(LIB.svoo_b200_cocluster_rows(
        q.data_ptr(), k.data_ptr(), qi_ptr, ki_ptr, BH, N, head_rows, D, QC, KC, int(iters),
        c.qlabels.data_ptr(), c.klabels.data_ptr(), c.qcentroids.data_ptr(), c.kcentroids.data_ptr(),
        c.qsizes.data_ptr(), c.ksizes.data_ptr(), c.q_sorted_idx.data_ptr(), c.q_offsets.data_ptr(),
        c.k_sorted_idx.data_ptr(), c.k_offsets.data_ptr(), ws.data_ptr(), ws.numel(), _stream()), "cocluster")
    return c


def cocluster_assign(x: torch.Tensor, form_centroids: torch.Tensor, own_centroids: torch.Tensor) -> torch.Tensor:
    """int32 labels [BH, N] of tokens x among own_centroids, profiles formed over form_centroids."""
    _need_cuda(x, form_centroids, own_centroids)
    BH, N, D = _tokens(x)
    K, J = form_centroids.shape[1], own_centroids.shape[1]
    labels = torch.empty(BH, N, dtype=torch.int32, device=x.device)
    ws = workspace(x.device, BH, N, K, J)
    check(LIB.svoo_b200_cocluster_assign(x.data_ptr(), form_centroids.data_ptr(), own_centroids.data_ptr(), BH, N, D,
                                         K, J, labels.data_ptr(), ws.data_ptr(), ws.numel(), _stream()),
          "cocluster_assign")
    return labels


def euclid_assign(x: torch.Tensor, centroids: torch.Tensor) -> torch.Tensor:
    """int32 labels [BH, N]: the nearest centroid of every token in Euclidean distance."""
    _need_cuda(x, centroids)
    BH, N, D = _tokens(x)
    K = centroids.shape[1]
    if centroids.shape != (BH, K, D) or centroids.dtype != x.dtype:
        raise ValueError("centroids must be bf16 [BH, K, 128]")
    labels = torch.empty(BH, N, dtype=torch.int32, device=x.device)
    ws = workspace(x.device, BH, N, K, K)
    check(LIB.svoo_b200_euclid_assign(x.data_ptr(), centroids.data_ptr(), BH, N, D, K, labels.data_ptr(), ws.data_ptr(),
                                      ws.numel(), _stream()), "euclid_assign")
    return labels


def append_text_blocks(block_map_u8: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                       q_sorted_idx: torch.Tensor, k_sorted_idx: torch.Tensor, text: int, prompt: int):
    """Map, offsets and row indices of a joint-attention layer whose `text` text rows follow the
    clustered video rows: (map [BH,QC+2,KC+2], q_off [BH,QC+3], k_off [BH,KC+3], q_idx, k_idx [BH,N+text])."""
    _need_cuda(block_map_u8, q_offsets, k_offsets, q_sorted_idx, k_sorted_idx)
    BH, QC, KC = block_map_u8.shape
    N = q_sorted_idx.shape[1]
    dev = block_map_u8.device
    i32 = dict(dtype=torch.int32, device=dev)
    m = torch.empty(BH, QC + 2, KC + 2, dtype=torch.uint8, device=dev)
    qo, ko = torch.empty(BH, QC + 3, **i32), torch.empty(BH, KC + 3, **i32)
    qi, ki = torch.empty(BH, N + text, **i32), torch.empty(BH, N + text, **i32)
    src = block_map_u8.view(torch.uint8) if block_map_u8.dtype == torch.bool else block_map_u8
    check(LIB.svoo_b200_append_text_blocks(src.data_ptr(), q_offsets.data_ptr(), k_offsets.data_ptr(),
                                           q_sorted_idx.data_ptr(), k_sorted_idx.data_ptr(), BH, N, QC, KC, int(text),
                                           int(prompt), m.data_ptr(), qo.data_ptr(), ko.data_ptr(), qi.data_ptr(),
                                           ki.data_ptr(), _stream()), "append_text_blocks")
    return m, qo, ko, qi, ki


def sort_labels(labels: torch.Tensor, num_clusters: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Stable cluster-order permutation: (sorted_idx int32 [BH,N], offsets int32 [BH,K+1]).
    Labels must lie in [0, num_clusters)."""
    _need_cuda(labels)
    lab = labels.to(torch.int32).contiguous()
    BH, N = lab.shape
    idx = torch.empty_like(lab)
    off = torch.empty(BH, num_clusters + 1, dtype=torch.int32, device=lab.device)
    ws = workspace(lab.device, BH, N, num_clusters, num_clusters)
    check(LIB.svoo_b200_sort_labels(lab.data_ptr(), BH, N, num_clusters, idx.data_ptr(), off.data_ptr(),
                                    ws.data_ptr(), ws.numel(), _stream()), "sort_labels")
    return idx, off


def centroid_update(x: torch.Tensor, sorted_idx: torch.Tensor, offsets: torch.Tensor,
                    old_centroids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    _need_cuda(x, sorted_idx, offsets, old_centroids)
    BH, N, D = _tokens(x)
    K = old_centroids.shape[1]
    new = torch.empty_like(old_centroids)
    sizes = torch.empty(BH, K, dtype=torch.int32, device=x.device)
    ws = workspace(x.device, BH, N, K, K)
    check(LIB.svoo_b200_centroid_update(x.data_ptr(), sorted_idx.data_ptr(), offsets.data_ptr(),
                                        old_centroids.data_ptr(), BH, N, D, K, new.data_ptr(), sizes.data_ptr(),
                                        ws.data_ptr(), ws.numel(), _stream()), "centroid_update")
    return new, sizes


def _head_rows(t: torch.Tensor, n: int) -> int:
    """Rows between consecutive heads of a [BH, >=n, 128] tensor whose rows are dense."""
    if t.dim() != 3 or t.shape[-1] != HEAD_DIM or t.stride(-1) != 1 or t.stride(1) != HEAD_DIM or t.shape[1] < n:
        raise ValueError("expected [BH, rows, 128] with dense rows")
    if t.shape[0] > 1 and t.stride(0) % HEAD_DIM:
        raise ValueError("head stride must be a whole number of rows")
    return t.stride(0) // HEAD_DIM if t.shape[0] > 1 else max(t.shape[1], n)


def permute(x: torch.Tensor, sorted_idx: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[bh, s] = x[bh, idx[bh, s]] for s < N = idx.shape[1]; x and out may be [BH, N, 128]
    views (leading rows) of longer per-head sequences."""
    N = sorted_idx.shape[1]
    BH = sorted_idx.shape[0]
    if not (x.is_cuda and sorted_idx.is_cuda and sorted_idx.is_contiguous() and x.dtype == torch.bfloat16):
        raise ValueError("permute needs CUDA bf16 tokens and a contiguous int32 index")
    y = torch.empty(BH, N, HEAD_DIM, dtype=x.dtype, device=x.device) if out is None else out
    check(LIB.svoo_b200_permute(x.data_ptr(), sorted_idx.data_ptr(), BH, N, HEAD_DIM, _head_rows(x, N),
                                _head_rows(y, N), y.data_ptr(), _stream()), "permute")
    return y


def inverse_permute(x: torch.Tensor, sorted_idx: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[bh, idx[bh, s]] = x[bh, s] for s < N = idx.shape[1]."""
    N = sorted_idx.shape[1]
    BH = sorted_idx.shape[0]
    if not (x.is_cuda and sorted_idx.is_cuda and sorted_idx.is_contiguous() and x.dtype == torch.bfloat16):
        raise ValueError("inverse_permute needs CUDA bf16 tokens and a contiguous int32 index")
    y = torch.empty(BH, N, HEAD_DIM, dtype=x.dtype, device=x.device) if out is None else out
    check(LIB.svoo_b200_inverse_permute(x.data_ptr(), sorted_idx.data_ptr(), BH, N, HEAD_DIM, _head_rows(x, N),
                                        _head_rows(y, N), y.data_ptr(), _stream()), "inverse_permute")
    return y


def block_map(qcentroids: torch.Tensor, kcentroids: torch.Tensor, ksizes: torch.Tensor, top_p: float,
              preserve: Sequence[int], cap: Sequence[int]) -> torch.Tensor:
    """uint8 [BH, QC, KC]; preserve / cap are per-head python ints (numbers of key clusters)."""
    _need_cuda(qcentroids, kcentroids, ksizes)
    BH, QC, D = qcentroids.shape
    KC = kcentroids.shape[1]
    if qcentroids.dtype != torch.bfloat16 or kcentroids.dtype != torch.bfloat16:
        raise ValueError("block_map needs bf16 centroids")
    if len(preserve) != BH or len(cap) != BH:
        raise ValueError("preserve and cap need one entry per head")
    out = torch.empty(BH, QC, KC, dtype=torch.uint8, device=qcentroids.device)
    arr = ctypes.c_int32 * BH
    ks = ksizes.to(torch.int32).contiguous()
    check(LIB.svoo_b200_block_map(qcentroids.data_ptr(), kcentroids.data_ptr(), ks.data_ptr(), BH, QC, KC, D,
                                  float(top_p), arr(*[int(v) for v in preserve]), arr(*[int(v) for v in cap]),
                                  out.data_ptr(), _stream()), "block_map")
    return out


def offsets_from_sizes(sizes: torch.Tensor) -> torch.Tensor:
    _need_cuda(sizes)
    s = sizes.to(torch.int32).contiguous()
    BH, K = s.shape
    off = torch.empty(BH, K + 1, dtype=torch.int32, device=s.device)
    check(LIB.svoo_b200_offsets_from_sizes(s.data_ptr(), BH, K, off.data_ptr(), _stream()), "offsets_from_sizes")
    return off


def sparse_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_map_u8: torch.Tensor,
                q_offsets: torch.Tensor, k_offsets: torch.Tensor, sm_scale: Optional[float] = None,
                out_row_idx: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                kernel: str = "tcgen05", peer_out=None, return_lse: bool = False):
    """Block-sparse attention over cluster-ordered q,k,v [BH,S,128].  With out_row_idx the
    result rows are scattered to their original positions (fused inverse permutation).
    kernel="simt" selects the mma.sync cross-check kernel.  peer_out = (peer pointer array,
    head id array, world, n_loc, H): the rows are stored into the ranks' sequence shards
    instead of a local tensor (svoo_b200_sparse_attn_push) and nothing is returned.
    return_lse: also return fp32 [BH, S], log2 of every row's softmax denominator (-inf for a row
    without keys), indexed like the output rows."""
    _need_cuda(q, k, v, block_map_u8, q_offsets, k_offsets)
    BH, S, D = _tokens(q)
    QC, KC = q_offsets.shape[1] - 1, k_offsets.shape[1] - 1
    if tuple(block_map_u8.shape) != (BH, QC, KC) or block_map_u8.dtype not in (torch.uint8, torch.bool):
        raise ValueError("block map must be uint8/bool [BH, QC, KC]")
    if kernel not in ("tcgen05", "simt"):
        raise ValueError("kernel must be 'tcgen05' or 'simt'")
    ws = workspace(q.device, BH, S, QC, KC)
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    ridx = 0 if out_row_idx is None else out_row_idx.data_ptr()
    if peer_out is not None:
        if kernel != "tcgen05":
            raise ValueError("peer stores need the tcgen05 kernel")
        ptrs, heads, world, n_loc, H = peer_out
        rc = LIB.svoo_b200_sparse_attn_push(q.data_ptr(), k.data_ptr(), v.data_ptr(), block_map_u8.data_ptr(),
                                            q_offsets.data_ptr(), k_offsets.data_ptr(), BH, S, D, QC, KC, scale, ptrs,
                                            heads, world, n_loc, H, ridx, ws.data_ptr(), ws.numel(), _stream())
        check(rc, "sparse_attn_push")
        return None
    y = torch.empty_like(q) if out is None else out
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), block_map_u8.data_ptr(), q_offsets.data_ptr(),
            k_offsets.data_ptr(), BH, S, D, QC, KC, scale, y.data_ptr())
    if kernel == "tcgen05":
        lse = torch.empty(BH, S, dtype=torch.float32, device=q.device) if return_lse else None
        rc = LIB.svoo_b200_sparse_attn(*head, ridx, 0 if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(),
                                       _stream())
        check(rc, "sparse_attn")
        return (y, lse) if return_lse else y
    if return_lse:
        raise ValueError("the log-sum-exp output needs the tcgen05 kernel")
    check(LIB.svoo_b200_sparse_attn_simt(*head, ridx, ws.data_ptr(), ws.numel(), _stream()), "sparse_attn")
    return y


@functools.lru_cache(maxsize=None)
def _all_heads(H: int):
    return (ctypes.c_int32 * H)(*range(H))


def token_major(out: torch.Tensor):
    """`peer_out` for sparse_attn / sparse_attn_ear that stores the rows of all H <= 128 heads into the local
    tensor out [1, S, H, 128]."""
    _, S, H, _ = out.shape
    return (ctypes.c_void_p * 1)(out.data_ptr()), _all_heads(H), 1, S, H


def attention_status(device: torch.device, BH: int, S: int, QC: int, KC: int) -> int:
    """Status word of the last svoo_b200_sparse_attn call that used this device's cached
    workspace with these sizes (synchronises).  0 = every CTA completed; non-zero = a CTA gave
    up on a bounded barrier wait and left its rows unwritten."""
    off = ctypes.c_int64(0)
    check(LIB.svoo_b200_status_offset(BH, S, QC, KC, ctypes.byref(off)), "status_offset")
    ws = workspace(device, BH, S, QC, KC)
    return int(ws[off.value:off.value + 4].view(torch.int32).item())


def cluster_status(device: torch.device, BH: int, N: int, QC: int, KC: int) -> int:
    """Same as attention_status for the assignment kernel of the last cocluster /
    cocluster_assign call (status word 1)."""
    off = ctypes.c_int64(0)
    check(LIB.svoo_b200_status_offset(BH, N, QC, KC, ctypes.byref(off)), "status_offset")
    ws = workspace(device, BH, N, QC, KC)
    return int(ws[off.value + 4:off.value + 8].view(torch.int32).item())


def qk_prep(x: torch.Tensor, heads: int, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
            cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The producer of the path's inputs in one pass: x [S, H*128] bf16 (a projection output) ->
    [H, S, 128] with the RMS norm over all H*128 columns (weight [H*128], any float dtype),
    the interleaved-pair rotary embedding (cos, sin [S, 128], the full-width tables; even cos and
    odd sin entries are used) and the head transpose.  weight / cos None skip that part (V)."""
    _need_cuda(x)
    if x.dim() != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous() or x.shape[1] != heads * 128:
        raise ValueError("x must be contiguous bf16 [S, H*128]")
    S = x.shape[0]
    w = None if weight is None else weight.detach().to(device=x.device, dtype=torch.float32).contiguous()
    if w is not None and w.numel() != heads * 128:
        raise ValueError("weight must have H*128 entries")
    c = s_ = None
    if cos is not None:
        c = cos.to(device=x.device, dtype=torch.float32).reshape(S, 128).contiguous()
        s_ = sin.to(device=x.device, dtype=torch.float32).reshape(S, 128).contiguous()
    out = torch.empty(heads, S, 128, dtype=torch.bfloat16, device=x.device)
    check(LIB.svoo_b200_qk_prep(x.data_ptr(), 0 if w is None else w.data_ptr(), float(eps), 0 if c is None else c.data_ptr(),
                                0 if s_ is None else s_.data_ptr(), S, heads, 128, out.data_ptr(), _stream()), "qk_prep")
    return out


def qk_prep_heads(x: torch.Tensor, heads: int, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                  cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, rope_rows: Optional[int] = None,
                  out: Optional[torch.Tensor] = None, out_row0: int = 0) -> torch.Tensor:
    """HunyuanVideo's producer in one pass: x [S, H*128] bf16 -> rows [out_row0, out_row0 + S) of
    out [H, rows, 128] with the RMS norm over the 128 values of every (token, head) (weight [128]),
    the interleaved-pair rotary embedding of the first `rope_rows` tokens (cos, sin [>= rope_rows, 128]) and
    the head transpose.  weight / cos None skip that part."""
    _need_cuda(x)
    if x.dim() != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous() or x.shape[1] != heads * 128:
        raise ValueError("x must be contiguous bf16 [S, H*128]")
    S = x.shape[0]
    w = None if weight is None else weight.detach().to(device=x.device, dtype=torch.float32).contiguous()
    if w is not None and w.numel() != 128:
        raise ValueError("weight must have 128 entries")
    rr = 0
    c = s_ = None
    if cos is not None:
        rr = S if rope_rows is None else int(rope_rows)
        c = cos.to(device=x.device, dtype=torch.float32).reshape(-1, 128).contiguous()
        s_ = sin.to(device=x.device, dtype=torch.float32).reshape(-1, 128).contiguous()
        if c.shape[0] < rr or s_.shape[0] < rr:
            raise ValueError("cos / sin need at least rope_rows rows")
    if out is None:
        out = torch.empty(heads, out_row0 + S, 128, dtype=torch.bfloat16, device=x.device)
    if out.dim() != 3 or out.shape[0] != heads or out.shape[2] != 128 or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("out must be contiguous bf16 [H, rows, 128]")
    check(LIB.svoo_b200_qk_prep_heads(x.data_ptr(), 0 if w is None else w.data_ptr(), float(eps),
                                      0 if c is None else c.data_ptr(), 0 if s_ is None else s_.data_ptr(), S, heads, 128, rr,
                                      out.data_ptr(), out.shape[1], int(out_row0), _stream()), "qk_prep_heads")
    return out


def layer(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_init_idx: torch.Tensor, k_init_idx: torch.Tensor,
          iters: int, top_p: float, preserve: Sequence[int], cap: Sequence[int],
          sm_scale: Optional[float] = None, text: int = 0, prompt: int = 0) -> torch.Tensor:
    """The whole layer through the single C entry point svoo_b200_layer: q, k, v [BH, S, 128] bf16
    in token order -> out [BH, S, 128]; the last `text` rows of every head are text tokens, of
    which the first `prompt` are the prompt.  Intermediates live in a scratch block that is
    released with the returned tensor's call frame; use the separate ops when they are needed."""
    _need_cuda(q, k, v, q_init_idx, k_init_idx)
    BH, S, D = _tokens(q)
    QC, KC = q_init_idx.shape[-1], k_init_idx.shape[-1]
    if len(preserve) != BH or len(cap) != BH:
        raise ValueError("preserve and cap need one entry per head")
    nbytes = ctypes.c_int64(0)
    check(LIB.svoo_b200_layer_scratch_bytes(BH, S, QC, KC, int(text), ctypes.byref(nbytes)), "layer_scratch_bytes")
    scratch = torch.empty(nbytes.value, dtype=torch.uint8, device=q.device)
    ws = workspace(q.device, BH, S, QC + 2, KC + 2) if text else workspace(q.device, BH, S, QC, KC)
    out = torch.empty_like(q)
    arr = ctypes.c_int32 * BH
    qi, ki = q_init_idx.to(torch.int32).contiguous(), k_init_idx.to(torch.int32).contiguous()
    check(LIB.svoo_b200_layer(q.data_ptr(), k.data_ptr(), v.data_ptr(), qi.data_ptr(), ki.data_ptr(), BH, S, D, QC, KC,
                              int(iters), float(top_p), arr(*[int(x) for x in preserve]), arr(*[int(x) for x in cap]),
                              D ** -0.5 if sm_scale is None else float(sm_scale), int(text), int(prompt), out.data_ptr(),
                              scratch.data_ptr(), scratch.numel(), ws.data_ptr(), ws.numel(), _stream()), "layer")
    return out


# ----------------------------------------------------------------------------------------------
# Error-aware routing (EAR)
# ----------------------------------------------------------------------------------------------
_ear_workspaces = {}


def ear_workspace(device: torch.device, BH: int, N: int, QC: int, KC: int) -> torch.Tensor:
    """Cached scratch of the EAR calls (one per device and stream); it carries the value statistics
    from ear_value_centroids to ear_block_scores."""
    need, _ = _ear_sizes(BH, N, QC, KC)
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    ws = _ear_workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        _ear_workspaces[key] = ws
    return ws


def _ear_sizes(BH, N, QC, KC):
    need, status = ctypes.c_int64(0), ctypes.c_int64(0)
    check(LIB.svoo_b200_ear_workspace_bytes(BH, N, QC, KC, ctypes.byref(need), ctypes.byref(status)), "ear_workspace_bytes")
    return need.value, status.value


def ear_value_centroids(v_perm: torch.Tensor, k_offsets: torch.Tensor, QC: int, out: Optional[torch.Tensor] = None):
    """Mean value row of every key cluster, bf16 [BH, KC, 128] (written into `out` when given, e.g. the
    centroid rows of an extended V tensor); the per-token statistics the block scores need stay in
    the EAR scratch of this device and stream."""
    _need_cuda(v_perm, k_offsets)
    BH, N, D = _tokens(v_perm)
    KC = k_offsets.shape[1] - 1
    vc = torch.empty(BH, KC, HEAD_DIM, dtype=torch.bfloat16, device=v_perm.device) if out is None else out
    ws = ear_workspace(v_perm.device, BH, N, QC, KC)
    check(LIB.svoo_b200_ear_value_centroids(v_perm.data_ptr(), k_offsets.data_ptr(), BH, N, D, QC, KC, vc.data_ptr(),
                                            ws.data_ptr(), ws.numel(), _stream()), "ear_value_centroids")
    return vc


def ear_block_scores(qcentroids: torch.Tensor, kcentroids: torch.Tensor, k_perm: torch.Tensor, q_offsets: torch.Tensor,
                     k_offsets: torch.Tensor, gamma: float):
    """(centroid logits, log-efficiency scores), fp32 [BH, QC, KC]; after ear_value_centroids on this
    device and stream."""
    _need_cuda(qcentroids, kcentroids, k_perm, q_offsets, k_offsets)
    BH, N, D = _tokens(k_perm)
    QC, KC = q_offsets.shape[1] - 1, k_offsets.shape[1] - 1
    if qcentroids.dtype != torch.bfloat16 or kcentroids.dtype != torch.bfloat16:
        raise ValueError("ear_block_scores needs bf16 centroids")
    clog = torch.empty(BH, QC, KC, dtype=torch.float32, device=k_perm.device)
    scores = torch.empty_like(clog)
    ws = ear_workspace(k_perm.device, BH, N, QC, KC)
    check(LIB.svoo_b200_ear_block_scores(qcentroids.contiguous().data_ptr(), kcentroids.contiguous().data_ptr(),
                                         k_perm.data_ptr(), q_offsets.data_ptr(), k_offsets.data_ptr(), BH, N, D, QC, KC,
                                         float(gamma), clog.data_ptr(), scores.data_ptr(), ws.data_ptr(), ws.numel(),
                                         _stream()), "ear_block_scores")
    return clog, scores


def ear_select_blocks(c_logits: torch.Tensor, scores: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                      top_p: float, preserve: Sequence[int], budget_preserve: Sequence[int]) -> torch.Tensor:
    """uint8 [BH, QC, KC]; preserve / budget_preserve are per-head python ints (numbers of key clusters)."""
    _need_cuda(c_logits, scores, q_offsets, k_offsets)
    BH, QC, KC = c_logits.shape
    if len(preserve) != BH or len(budget_preserve) != BH:
        raise ValueError("preserve and budget_preserve need one entry per head")
    if c_logits.dtype != torch.float32 or scores.dtype != torch.float32 or tuple(scores.shape) != (BH, QC, KC):
        raise ValueError("c_logits and scores must be fp32 [BH, QC, KC]")
    out = torch.empty(BH, QC, KC, dtype=torch.uint8, device=c_logits.device)
    arr = ctypes.c_int32 * BH
    check(LIB.svoo_b200_ear_select_blocks(c_logits.contiguous().data_ptr(), scores.contiguous().data_ptr(),
                                          q_offsets.data_ptr(), k_offsets.data_ptr(), BH, QC, KC, float(top_p),
                                          arr(*[int(v) for v in preserve]), arr(*[int(v) for v in budget_preserve]),
                                          out.data_ptr(), _stream()), "ear_select_blocks")
    return out


def sparse_attn_ear(q: torch.Tensor, k_ext: torch.Tensor, v_ext: torch.Tensor, block_map_u8: torch.Tensor,
                    q_offsets: torch.Tensor, k_offsets: torch.Tensor, sm_scale: Optional[float] = None,
                    out_row_idx: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, peer_out=None):
    """EAR forward: q [BH,S,128] in cluster order; k_ext, v_ext [BH*S + BH*KC, 128] = the cluster-ordered
    rows of all heads followed by the key / value centroid rows of all heads.  Output, out_row_idx, the
    log2-sum-exp and peer_out as in sparse_attn."""
    _need_cuda(q, k_ext, v_ext, block_map_u8, q_offsets, k_offsets)
    BH, S, D = _tokens(q)
    QC, KC = q_offsets.shape[1] - 1, k_offsets.shape[1] - 1
    if tuple(block_map_u8.shape) != (BH, QC, KC) or block_map_u8.dtype not in (torch.uint8, torch.bool):
        raise ValueError("block map must be uint8/bool [BH, QC, KC]")
    for t in (k_ext, v_ext):
        if tuple(t.shape) != (BH * S + BH * KC, HEAD_DIM) or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError("k_ext and v_ext must be contiguous bf16 [BH*S + BH*KC, 128]")
    ws = ear_workspace(q.device, BH, S, QC, KC)
    if peer_out is not None:
        ptrs, heads, world, n_loc, H = peer_out
        check(LIB.svoo_b200_sparse_attn_ear_push(q.data_ptr(), k_ext.data_ptr(), v_ext.data_ptr(), block_map_u8.data_ptr(),
                                                 q_offsets.data_ptr(), k_offsets.data_ptr(), BH, S, D, QC, KC,
                                                 D ** -0.5 if sm_scale is None else float(sm_scale), ptrs, heads, world, n_loc,
                                                 H, 0 if out_row_idx is None else out_row_idx.data_ptr(), ws.data_ptr(),
                                                 ws.numel(), _stream()), "sparse_attn_ear_push")
        return None
    y = torch.empty_like(q) if out is None else out
    lse = torch.empty(BH, S, dtype=torch.float32, device=q.device) if return_lse else None
    check(LIB.svoo_b200_sparse_attn_ear(q.data_ptr(), k_ext.data_ptr(), v_ext.data_ptr(), block_map_u8.data_ptr(),
                                        q_offsets.data_ptr(), k_offsets.data_ptr(), BH, S, D, QC, KC,
                                        D ** -0.5 if sm_scale is None else float(sm_scale), y.data_ptr(),
                                        0 if out_row_idx is None else out_row_idx.data_ptr(),
                                        0 if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), _stream()),
          "sparse_attn_ear")
    return (y, lse) if return_lse else y


def ear_attention_status(device: torch.device, BH: int, S: int, QC: int, KC: int) -> int:
    """Status word of the last sparse_attn_ear on this device and stream (0 = no bounded wait expired)."""
    _, off = _ear_sizes(BH, S, QC, KC)
    ws = ear_workspace(device, BH, S, QC, KC)
    return int(ws[off:off + 4].view(torch.int32).item())


# ----------------------------------------------------------------------------------------------
# Token-wise operators: layer norm, 8-bit linear layers.  They run on the device of their tensors (the current
# stream of that device) and take their scratch from torch's allocator, call by call: a captured graph owns what
# it uses, and calls on different streams share nothing.
# ----------------------------------------------------------------------------------------------
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
E4M3 = torch.float8_e4m3fn
_E4M3_TYPE = 3
_ACTIVATIONS = {None: 0, "gelu": 1}


_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream      # what torch.cuda.current_stream(index).cuda_stream says, without its objects


def _device(*tensors: Optional[torch.Tensor]) -> int:
    """The index of the one CUDA device that all the tensors are on."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()
        if at < 0:
            raise ValueError("svoo_b200 ops need CUDA tensors; there is no CPU path")
        if index < 0:
            index = at
        elif at != index:
            raise ValueError("all tensors of a call must be on one device")
    return index


def refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Raises where a tensor carries a tangent of forward-mode differentiation: the kernels would drop it."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("svoo_b200 operators have no forward-mode gradient")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _norm_rows(x: torch.Tensor, what: str) -> Tuple[int, int, int, int]:
    """(batch, rows, batch stride, row stride) of a tensor [..., C] whose last dimension is dense: any layout with up to three
    dimensions, dense ones beyond that."""
    shape = x.shape
    dims = len(shape)
    if x.dtype not in TYPES:
        raise ValueError(f"{what} must be bf16, fp16 or fp32, got {x.dtype}")
    if dims < 1:
        raise ValueError(f"{what} needs at least one dimension")
    C = shape[-1]
    if x.is_contiguous():
        if dims == 3:
            return shape[0], shape[1], shape[1] * C, C
        return 1, x.numel() // C if C else 0, 0, C
    if dims > 3 or (C > 1 and x.stride(-1) != 1):
        raise ValueError(f"the last dimension of {what} must be dense, and all of them beyond three")
    if dims == 3:
        return shape[0], shape[1], x.stride(0), x.stride(1)
    return 1, shape[0], 0, x.stride(0)


def _norm_params(x: torch.Tensor, weight, bias, scale, shift):
    """Checks gain and offset against x: (gain, offset, strides of both per sample, type, whether gain means 1 + gain, whether
    there is one per sample)."""
    if scale is None and shift is None:
        if weight is None:
            if bias is not None:
                raise ValueError("bias needs weight, and shift needs scale")
            return None, None, 0, 0, torch.float32, False, False
        shape, dtype, C = weight.shape, weight.dtype, x.shape[-1]
        if len(shape) != 1 or shape[0] != C:
            raise ValueError(f"weight and bias must be [{C}], got {list(shape)}")
        gain, offset, plus_one, per_sample, gb, ob = weight, bias, False, False, 0, 0
    else:
        if weight is not None or bias is not None:
            raise ValueError("a layer norm takes weight and bias, or scale and shift, not both")
        if scale is None:
            raise ValueError("bias needs weight, and shift needs scale")
        shape, dtype, C = tuple(scale.shape), scale.dtype, x.shape[-1]
        B = x.shape[0] if x.dim() == 3 else 1
        if x.dim() > 3 or shape not in ((B, 1, C), (B, C), (1, 1, C), (1, C)):
            raise ValueError(f"scale and shift must be [B, 1, {C}] or [B, {C}] for an input [B, S, {C}], got {list(shape)}")
        gain, offset, plus_one = scale, shift, True
        per_sample = shape[0] == B and B > 1
        gb = scale.stride(0) if per_sample else 0
        ob = shift.stride(0) if per_sample and shift is not None else 0
    if dtype is not torch.float32 and dtype is not x.dtype:
        raise ValueError(f"parameters must be fp32 or of the input's type, got {dtype}")
    if offset is not None and (offset.dtype is not dtype or offset.shape != gain.shape):
        raise ValueError("both parameters must have one type and one shape")
    if C > 1 and (gain.stride(-1) != 1 or (offset is not None and offset.stride(-1) != 1)):
        raise ValueError("the last dimension of every parameter must be dense")
    return gain, offset, gb, ob, dtype, plus_one, per_sample


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
               return_stats: bool = False):
    """Layer norm over the last dimension (at most 16,384 columns) of x [..., C], bf16, fp16 or fp32: affine with weight and
    bias [C], modulated with 1 + scale and shift [B, 1, C] or [B, C] for x [B, S, C], or neither.  Parameters in fp32 or x's type.
    Statistics in 32 bits.  Returns y, dense and of x's type; with return_stats (y, mean, rstd), fp32 of the leading dimensions.
    Not differentiable by itself: see norm.layer_norm."""
    batch, rows, xb, xr = _norm_rows(x, "x")
    gain, offset, gb, ob, dtype, plus_one, _ = _norm_params(x, weight, bias, scale, shift)
    index = _device(x, gain, offset)
    if index != _current_device():
        with torch.cuda.device(index):
            return layer_norm(x, weight, bias, scale, shift, eps, return_stats)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = None
    if return_stats:
        mean, rstd = (x.new_empty(x.shape[:-1], dtype=torch.float32) for _ in range(2))
    check(LIB.svoo_b200_layer_norm(x.data_ptr(), TYPES[x.dtype], batch, rows, x.shape[-1], xb, xr, _ptr(gain), gb, _ptr(offset), ob,
                                   TYPES[dtype], plus_one, eps, y.data_ptr(), _ptr(mean), _ptr(rstd), _raw_stream(index)), "layer_norm")
    return (y, mean, rstd) if return_stats else y


@functools.lru_cache(maxsize=1024)
def _norm_workspace_bytes(batch: int, rows: int, C: int, per_sample: bool) -> int:
    need = ctypes.c_int64(0)
    check(LIB.svoo_b200_layer_norm_workspace_bytes(batch, rows, C, per_sample, ctypes.byref(need)), "layer_norm_backward")
    return need.value


def layer_norm_backward(grad: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, param_grads: bool = True):
    """Gradient of layer_norm at `grad` (y's shape and type): (dx, dgain, doffset), dgain and doffset of the shape and type of
    weight or scale (None without one, or without param_grads).  mean, rstd as layer_norm returned them.  The sums over the rows
    run in a fixed order: the same call gives the same bits."""
    batch, rows, xb, xr = _norm_rows(x, "x")
    if grad.shape != x.shape or grad.dtype != x.dtype:
        raise ValueError("the gradient must have the shape and type of x")
    _, _, db, dr = _norm_rows(grad, "the gradient")
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1] or not t.is_contiguous():
            raise ValueError("mean and rstd must be what layer_norm returned: contiguous fp32 of x's leading dimensions")
    gain, _, gb, _, dtype, plus_one, per_sample = _norm_params(x, weight, None, scale, None)
    C = x.shape[-1]
    index = _device(x, grad, mean, rstd, gain)
    if index != _current_device():
        with torch.cuda.device(index):
            return layer_norm_backward(grad, x, mean, rstd, weight, scale, param_grads)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dgain = doffset = ws = None
    ws_bytes = 0
    if param_grads and gain is not None:
        make = gain.new_zeros if batch == 0 else gain.new_empty
        dgain, doffset = make(gain.shape), make(gain.shape)
        ws_bytes = _norm_workspace_bytes(batch, rows, C, per_sample)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    check(LIB.svoo_b200_layer_norm_backward(grad.data_ptr(), db, dr, x.data_ptr(), TYPES[x.dtype], batch, rows, C, xb, xr,
                                            mean.data_ptr(), rstd.data_ptr(), _ptr(gain), gb, TYPES[dtype], plus_one, per_sample,
                                            dx.data_ptr(), _ptr(dgain), _ptr(doffset), _ptr(ws), ws_bytes, _raw_stream(index)),
          "layer_norm_backward")
    return dx, dgain, doffset


@dataclasses.dataclass
class Fp8Rows:
    """A matrix in e4m3 with one fp32 scale per 1 x 128 block: q [M, K], rows a multiple of 16 bytes apart; scale
    [ceil(K / 128), M], one row per block column."""
    q: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self):
        return self.q.shape

    def float(self) -> torch.Tensor:
        """The values it stands for, fp32 (plain torch)."""
        return self.q.float() * self.scale.t().repeat_interleave(128, 1)[:, :self.q.shape[1]]


@dataclasses.dataclass
class Fp8Blocks:
    """A matrix in e4m3 with one fp32 scale per 128 x 128 block: q [N, K], rows a multiple of 16 bytes apart; scale
    [ceil(N / 128), ceil(K / 128)].  qt, where present, is the transpose of q, for the gradient of the other operand."""
    q: torch.Tensor
    scale: torch.Tensor
    qt: Optional[torch.Tensor] = None

    @property
    def shape(self):
        return self.q.shape

    def transposed(self) -> "Fp8Blocks":
        if self.qt is None:
            raise ValueError("quantised without its transpose")
        return Fp8Blocks(self.qt, self.scale.t(), self.q)

    def float(self) -> torch.Tensor:
        """The values it stands for, fp32 (plain torch)."""
        N, K = self.q.shape
        return self.q.float() * self.scale.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def _matrix(x: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(rows, columns, row stride) of a matrix with dense rows."""
    if x.dim() != 2 or x.dtype not in TYPES:
        raise ValueError(f"{what} must be a bf16, fp16 or fp32 matrix, got {x.dtype} {tuple(x.shape)}")
    M, K = x.shape
    if K < 1 or (K > 1 and x.stride(1) != 1):
        raise ValueError(f"{what} needs dense rows of at least one column")
    return M, K, x.stride(0) if M > 1 else K


def _pad16(n: int) -> int:
    return (n + 15) & ~15


def _empty_e4m3(like: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    pitch = _pad16(cols)
    q = like.new_empty((rows, pitch), dtype=E4M3)
    return q if pitch == cols else q[:, :cols]


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """x [M, K] (bf16, fp16, fp32; dense rows) in e4m3, one scale max(amax / 448, 2^-126) per 1 x 128 block, values to the nearest.
    A block with a value that is not finite stands for NaN."""
    M, K, stride = _matrix(x, "x")
    index = _device(x)
    if index != _current_device():
        with torch.cuda.device(index):
            return quantize_rows(x)
    q = _empty_e4m3(x, M, K)
    scale = x.new_empty(((K + 127) // 128, M), dtype=torch.float32)
    check(LIB.svoo_b200_quantize_rows(x.data_ptr(), TYPES[x.dtype], M, K, stride, q.data_ptr(), _pad16(K), scale.data_ptr(), M,
                                      _raw_stream(index)), "quantize_rows")
    return Fp8Rows(q, scale)


def quantize_columns(x: torch.Tensor, column_sum_type: Optional[torch.dtype] = None):
    """The transpose of x [M, K] quantised along M: Fp8Rows of shape [K, M].  With column_sum_type also the sums of x's columns,
    [K] of that type, added in 32 bits in a fixed order: (rows, sums).  1 <= M <= 65,535 x 128."""
    M, K, stride = _matrix(x, "x")
    if M < 1:
        raise ValueError("quantize_columns needs at least one row")
    if column_sum_type is not None and column_sum_type not in TYPES:
        raise ValueError("column sums are bf16, fp16 or fp32")
    index = _device(x)
    if index != _current_device():
        with torch.cuda.device(index):
            return quantize_columns(x, column_sum_type)
    MB, pitch = (M + 127) // 128, (K + 3) // 4 * 4
    q = _empty_e4m3(x, K, M)
    scale = x.new_empty((MB, pitch), dtype=torch.float32)
    part = None if column_sum_type is None else x.new_empty((MB, K), dtype=torch.float32)
    stream = _raw_stream(index)
    check(LIB.svoo_b200_quantize_columns(x.data_ptr(), TYPES[x.dtype], M, K, stride, q.data_ptr(), _pad16(M), scale.data_ptr(), pitch,
                                         _ptr(part), stream), "quantize_columns")
    rows = Fp8Rows(q, scale[:, :K])
    if part is None:
        return rows
    sums = x.new_empty(K, dtype=column_sum_type)
    check(LIB.svoo_b200_column_sum(part.data_ptr(), MB, K, sums.data_ptr(), TYPES[column_sum_type], stream), "column_sum")
    return rows, sums


def quantize_both(x: torch.Tensor, column_sum_type: Optional[torch.dtype] = None):
    """(quantize_rows(x), quantize_columns(x)) from one reading of x [M, K], M >= 1; with column_sum_type also the sums of the
    columns, as quantize_columns gives them."""
    M, K, stride = _matrix(x, "x")
    if M < 1:
        raise ValueError("quantize_both needs at least one row")
    if column_sum_type is not None and column_sum_type not in TYPES:
        raise ValueError("column sums are bf16, fp16 or fp32")
    index = _device(x)
    if index != _current_device():
        with torch.cuda.device(index):
            return quantize_both(x, column_sum_type)
    KB, MB, pitch = (K + 127) // 128, (M + 127) // 128, (K + 3) // 4 * 4
    q, qt = _empty_e4m3(x, M, K), _empty_e4m3(x, K, M)
    scale, scale_t = x.new_empty((KB, M), dtype=torch.float32), x.new_empty((MB, pitch), dtype=torch.float32)
    part = None if column_sum_type is None else x.new_empty((MB, K), dtype=torch.float32)
    stream = _raw_stream(index)
    check(LIB.svoo_b200_quantize_both(x.data_ptr(), TYPES[x.dtype], M, K, stride, q.data_ptr(), _pad16(K), scale.data_ptr(), M, qt.data_ptr(),
                                      _pad16(M), scale_t.data_ptr(), pitch, _ptr(part), stream), "quantize_both")
    rows, columns = Fp8Rows(q, scale), Fp8Rows(qt, scale_t[:, :K])
    if part is None:
        return rows, columns
    sums = x.new_empty(K, dtype=column_sum_type)
    check(LIB.svoo_b200_column_sum(part.data_ptr(), MB, K, sums.data_ptr(), TYPES[column_sum_type], stream), "column_sum")
    return rows, columns, sums


def quantize_blocks(w: torch.Tensor, transposed: bool = False) -> Fp8Blocks:
    """w [N, K] in e4m3, one scale per 128 x 128 block; `transposed` keeps the transpose of the bytes too."""
    N, K, stride = _matrix(w, "w")
    if N < 1:
        raise ValueError("quantize_blocks needs at least one row")
    index = _device(w)
    if index != _current_device():
        with torch.cuda.device(index):
            return quantize_blocks(w, transposed)
    q = _empty_e4m3(w, N, K)
    qt = _empty_e4m3(w, K, N) if transposed else None
    scale = w.new_empty(((N + 127) // 128, (K + 127) // 128), dtype=torch.float32)
    check(LIB.svoo_b200_quantize_blocks(w.data_ptr(), TYPES[w.dtype], N, K, stride, q.data_ptr(), _pad16(K), _ptr(qt), _pad16(N),
                                        scale.data_ptr(), _raw_stream(index)), "quantize_blocks")
    return Fp8Blocks(q, scale, qt)


def _e4m3_operand(q: torch.Tensor, scale: torch.Tensor, scale_shape, what: str) -> int:
    """Pitch of an e4m3 matrix; checks it and the shape of its scales."""
    if q.dtype is not E4M3 or q.dim() != 2 or q.shape[1] < 1 or (q.shape[1] > 1 and q.stride(1) != 1):
        raise ValueError(f"{what} must be an e4m3 matrix with dense rows")
    pitch = q.stride(0) if q.shape[0] > 1 else _pad16(q.shape[1])
    if pitch % 16 or pitch < q.shape[1] or q.data_ptr() % 16:
        raise ValueError(f"{what} needs rows a multiple of 16 bytes apart and a 16-byte aligned start")
    if scale.dtype is not torch.float32 or scale.shape != scale_shape:
        raise ValueError(f"the scales of {what} must be fp32 {list(scale_shape)}, got {scale.dtype} {list(scale.shape)}")
    return pitch


def _product_output(like: torch.Tensor, M: int, N: int, bias, activation, out_dtype):
    """Checks bias, activation and type; (out, its scales or None, pitch, type number)."""
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'gelu'")
    if bias is not None and (bias.dtype not in TYPES or bias.dim() != 1 or bias.shape[0] != N or (N > 1 and bias.stride(0) != 1)):
        raise ValueError(f"bias must be a dense [{N}] of bf16, fp16 or fp32")
    if out_dtype is E4M3:
        return _empty_e4m3(like, M, N), like.new_empty(((N + 127) // 128, M), dtype=torch.float32), _pad16(N), _E4M3_TYPE
    if out_dtype not in TYPES:
        raise ValueError("out_dtype must be bf16, fp16, fp32 or float8_e4m3fn")
    return like.new_empty((M, N), dtype=out_dtype), None, N, TYPES[out_dtype]


def mm_fp8(a: Fp8Rows, b, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           out_dtype: torch.dtype = torch.bfloat16):
    """act(a b^T + bias), sums in 32 bits: a Fp8Rows [M, K]; b Fp8Blocks [N, K], or Fp8Rows [N, K], its scales on 16 bytes and their
    rows a multiple of four apart, as quantize_columns leaves them (then neither of the next two); bias [N], bf16, fp16 or fp32;
    activation None or "gelu" (its tanh formula).  out_dtype bf16, fp16, fp32, or float8_e4m3fn for the 32-bit results quantised in
    1 x 128 blocks, an Fp8Rows, ready to be the next product's a."""
    M, K = a.q.shape
    N = b.q.shape[0]
    KB = (K + 127) // 128
    rows = isinstance(b, Fp8Rows)
    if b.q.shape[1] != K or N < 1:
        raise ValueError(f"a [{M}, {K}] and b {list(b.q.shape)} do not sum over the same length")
    if rows and (out_dtype is E4M3 or activation is not None or bias is not None):
        raise ValueError("a product of two Fp8Rows takes no bias or activation and gives no e4m3 output")
    ap = _e4m3_operand(a.q, a.scale, (KB, M), "a")
    bp = _e4m3_operand(b.q, b.scale, (KB, N) if rows else ((N + 127) // 128, KB), "b")
    if M > 1 and a.scale.stride(1) != 1:
        raise ValueError("the scales of a must be dense along the rows of a")
    sn, sk = (1, b.scale.stride(0)) if rows else b.scale.stride()
    if rows and KB == 1:
        sk = (N + 3) // 4 * 4
    if rows and (N > 1 and b.scale.stride(1) != 1 or sk % 4 or sk < N or b.scale.data_ptr() % 16):
        raise ValueError("the scales of b must be dense along its rows, with a 16-byte aligned start and pitch")
    index = _device(a.q, a.scale, b.q, b.scale, bias)
    if index != _current_device():
        with torch.cuda.device(index):
            return mm_fp8(a, b, bias, activation, out_dtype)
    out, out_scale, pitch, kind = _product_output(a.q, M, N, bias, activation, out_dtype)
    check(LIB.svoo_b200_mm_fp8(a.q.data_ptr(), ap, a.scale.data_ptr(), a.scale.stride(0) if KB > 1 else M, b.q.data_ptr(), bp,
                               b.scale.data_ptr(), sn, sk, rows, _ptr(bias), 0 if bias is None else TYPES[bias.dtype], M, N, K,
                               _ACTIVATIONS[activation], out.data_ptr(), kind, pitch, _ptr(out_scale), M, _raw_stream(index)), "mm_fp8")
    return out if out_scale is None else Fp8Rows(out, out_scale)


def linear_fp8(x: torch.Tensor, w: Fp8Blocks, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
               out_dtype: Optional[torch.dtype] = None):
    """mm_fp8(quantize_rows(x), w, bias, activation, out_dtype or x's type) in one call: x [M, K] (bf16, fp16, fp32; dense
    rows).  Few rows (8, or 16 of up to 4,096 columns) are one launch, whose 32-bit sums run in another order than mm_fp8's."""
    M, K, stride = _matrix(x, "x")
    q, scale = w.q, w.scale
    N = q.shape[0]
    KB = (K + 127) // 128
    if q.shape[1] != K or N < 1:
        raise ValueError(f"x [{M}, {K}] and w {list(q.shape)} do not sum over the same length")
    wp = _e4m3_operand(q, scale, ((N + 127) // 128, KB), "w")
    index = _device(x, q, scale, bias)
    if index != _current_device():
        with torch.cuda.device(index):
            return linear_fp8(x, w, bias, activation, out_dtype)
    out, out_scale, pitch, kind = _product_output(x, M, N, bias, activation, out_dtype or x.dtype)
    ws, ws_bytes = None, 0                                  # as svoo_b200_linear_fp8_workspace_bytes
    if M > 16 or (M > 8 and K > 4096) or out_scale is not None:
        ws_bytes = (M * _pad16(K) + 255) // 256 * 256 + KB * M * 4
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    check(LIB.svoo_b200_linear_fp8(x.data_ptr(), TYPES[x.dtype], M, K, stride, q.data_ptr(), wp, scale.data_ptr(), scale.stride(0),
                                   scale.stride(1), _ptr(bias), 0 if bias is None else TYPES[bias.dtype], N, _ACTIVATIONS[activation],
                                   out.data_ptr(), kind, pitch, _ptr(out_scale), M, _ptr(ws), ws_bytes, _raw_stream(index)), "linear_fp8")
    return out if out_scale is None else Fp8Rows(out, out_scale)


@functools.lru_cache(maxsize=1024)
def _train_bytes(M: int, N: int, K: int, keep_x: bool, keep_w: bool) -> Tuple[int, int, int]:
    need = (ctypes.c_int64 * 3)()
    check(LIB.svoo_b200_linear_train_bytes(M, N, K, keep_x, keep_w, need), "linear_train")
    return tuple(need)


def linear_train_forward(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, keep_x_grad: bool = True,
                         keep_w_grad: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(x w^T + bias, saved) of a layer in training: x [M, K], M >= 1, and w [N, K], both quantised in the call (quantize_rows,
    quantize_blocks), results as mm_fp8 gives them; `saved`, bytes, is what linear_train_backward needs for the gradient of x and of w."""
    M, K, x_row = _matrix(x, "x")
    N, KW, w_row = _matrix(w, "w")
    if K != KW or M < 1 or N < 1:
        raise ValueError(f"x {[M, K]} and w {[N, KW]} do not sum over the same length, or have no rows")
    if bias is not None and (bias.dtype not in TYPES or bias.dim() != 1 or bias.shape[0] != N or (N > 1 and bias.stride(0) != 1)):
        raise ValueError(f"bias must be a dense [{N}] of bf16, fp16 or fp32")
    index = _device(x, w, bias)
    if index != _current_device():
        with torch.cuda.device(index):
            return linear_train_forward(x, w, bias, keep_x_grad, keep_w_grad)
    saved_bytes, scratch_bytes, _ = _train_bytes(M, N, K, keep_x_grad, keep_w_grad)
    y = x.new_empty((M, N))
    saved, scratch = x.new_empty(saved_bytes, dtype=torch.uint8), x.new_empty(scratch_bytes, dtype=torch.uint8)
    check(LIB.svoo_b200_linear_train_forward(x.data_ptr(), TYPES[x.dtype], M, K, x_row, w.data_ptr(), TYPES[w.dtype], N, w_row, _ptr(bias),
                                             0 if bias is None else TYPES[bias.dtype], keep_x_grad, keep_w_grad, y.data_ptr(),
                                             saved.data_ptr(), saved_bytes, scratch.data_ptr(), scratch_bytes, _raw_stream(index)),
          "linear_train_forward")
    return y, saved


def linear_train_backward(grad: torch.Tensor, saved: torch.Tensor, K: int, keep_x_grad: bool = True, keep_w_grad: bool = True,
                          x_grad: bool = True, w_dtype: Optional[torch.dtype] = None, bias_dtype: Optional[torch.dtype] = None):
    """(dx or None, dw or None, db or None) of linear_train_forward at grad [M, N] (the type of its result): dx with x_grad, dw and db
    of w_dtype and bias_dtype where those are given.  K and the keep flags as in the forward call."""
    M, N, row = _matrix(grad, "the gradient")
    if (x_grad and not keep_x_grad) or (w_dtype is not None and not keep_w_grad):
        raise ValueError("the forward call did not keep what this gradient needs")
    if not all(t is None or t in TYPES for t in (w_dtype, bias_dtype)):
        raise ValueError("gradients are bf16, fp16 or fp32")
    saved_bytes, _, scratch_bytes = _train_bytes(M, N, K, keep_x_grad, keep_w_grad)
    if saved.dtype is not torch.uint8 or saved.dim() != 1 or saved.shape[0] != saved_bytes:
        raise ValueError("saved is not of a forward call with these sizes")
    index = _device(grad, saved)
    if index != _current_device():
        with torch.cuda.device(index):
            return linear_train_backward(grad, saved, K, keep_x_grad, keep_w_grad, x_grad, w_dtype, bias_dtype)
    dx = grad.new_empty((M, K)) if x_grad else None
    dw = None if w_dtype is None else grad.new_empty((N, K), dtype=w_dtype)
    db = None if bias_dtype is None else grad.new_empty(N, dtype=bias_dtype)
    scratch = grad.new_empty(scratch_bytes, dtype=torch.uint8)
    check(LIB.svoo_b200_linear_train_backward(grad.data_ptr(), TYPES[grad.dtype], M, N, K, row, saved.data_ptr(), saved_bytes, keep_x_grad,
                                              keep_w_grad, _ptr(dx), _ptr(dw), TYPES.get(w_dtype, 0), _ptr(db), TYPES.get(bias_dtype, 0),
                                              scratch.data_ptr(), scratch_bytes, _raw_stream(index)), "linear_train_backward")
    return dx, dw, db


def linear_status(device: torch.device) -> int:
    """Status word of the layer norms and 8-bit products on this device (synchronises): 0, or 1 once a kernel has given up on a
    bounded wait and left rows unwritten.  It stays 1."""
    with torch.cuda.device(device):
        out = torch.zeros(1, dtype=torch.int32, device="cuda")
        check(LIB.svoo_b200_linear_status(out.data_ptr(), _stream()), "linear_status")
        return int(out.item())
