"""Host-side mirror of ``nntile.layer.Sdpa`` for the path (reference:
wrappers/python/nntile/layer/sdpa.py).

Tensors are torch CUDA buffers holding NNTile's Fortran-order arrays: an NNTile
tensor of shape [head, seq, batch, group, kv_heads] is a contiguous torch tensor
of shape (kv_heads, group, batch, seq, head).  ``from_fortran`` / ``to_fortran``
convert from and to numpy Fortran arrays (bf16 as uint16 bit patterns).

``Sdpa`` issues the same operations in the same order as the reference layer:
the unfused chain (gemm -> mask_scalar -> maxsumexp -> softmax_inplace -> gemm
and its backward, sdpa.py:407-455, 595-698) or the fused tile tasks (fill/clear
prologue + flash forward, flash backward, sdpa.py:533-593) with the reference's
tile loops run by the C library.
"""
from __future__ import annotations

import ctypes
import itertools
import math
import os
import warnings

import numpy as np
import torch

from . import _lib, build, ops


def _load_paged_torch():
    """The paged calls without the interpreter between the tensors and the library; what the
    module does not take (and every mistake) goes the way through ops, as everything does when
    it was not built.  One that was built and does not load is said."""
    try:
        from . import _paged_torch
        return _paged_torch
    except ImportError as e:
        if os.path.exists(build.TORCH_MODULE):
            warnings.warn(f"{build.TORCH_MODULE} does not load ({e}): paged calls take longer on the "
                          "host. Build it again: python -m nntile_b200.build", RuntimeWarning)
        return None


_paged_torch = _load_paged_torch()


def from_fortran(arr: np.ndarray, device="cuda") -> torch.Tensor:
    """numpy Fortran array (float32, float16, or uint16 = bf16 bits) -> torch buffer."""
    a = np.asfortranarray(arr)
    if a.dtype == np.uint16:
        return torch.from_numpy(a.T.view(np.int16).copy()).view(torch.bfloat16).to(device)
    if a.dtype == np.bool_:
        return torch.from_numpy(a.T.copy()).to(device)
    return torch.from_numpy(a.T.copy()).to(device)


def to_fortran(t: torch.Tensor) -> np.ndarray:
    t = t.detach().cpu().contiguous()
    if t.dtype == torch.bfloat16:
        return np.asfortranarray(t.view(torch.int16).numpy().view(np.uint16).T)
    return np.asfortranarray(t.numpy().T)


def sdpa_scale(head_size: int) -> float:
    """sdpa.py:149."""
    return float(np.float32(1.0)/np.sqrt(np.float32(head_size)))


class TiledBuffer:
    """A tensor cut into separately stored Fortran-order tiles, the storage model
    of nntile::tensor::Tensor (include/nntile/tensor/tensor.hh).  `shape` and
    `basetile` are in NNTile (Fortran) order."""

    def __init__(self, full: torch.Tensor, basetile):
        self.shape = tuple(reversed(full.shape))
        self.basetile = tuple(int(b) for b in basetile)
        self.grid = tuple(-(-s//b) for s, b in zip(self.shape, self.basetile))
        self.dtype = full.dtype
        self.tiles = []
        # Fortran order of the tile grid: first index fastest
        for idx in itertools.product(*(range(g) for g in reversed(self.grid))):
            idx = tuple(reversed(idx))
            self.tiles.append(full[self._slices(idx)].contiguous())

    def _slices(self, idx):
        sl = [slice(i*b, min((i + 1)*b, s)) for i, b, s in zip(idx, self.basetile, self.shape)]
        return tuple(reversed(sl))

    def pointers(self):
        arr = (ctypes.c_void_p*len(self.tiles))(*[t.data_ptr() for t in self.tiles])
        return arr

    def gather(self) -> torch.Tensor:
        out = torch.empty(tuple(reversed(self.shape)), dtype=self.dtype,
                          device=self.tiles[0].device)
        for n, idx in enumerate(itertools.product(*(range(g) for g in reversed(self.grid)))):
            out[self._slices(tuple(reversed(idx)))] = self.tiles[n]
        return out


def _i64arr(vals):
    return (ctypes.c_int64*len(vals))(*[int(v) for v in vals])


def _tensor_call(name, shape5, base5, tiled, scratch_holder=None):
    """Run one tensor-level C entry point on lists of TiledBuffer."""
    lib = _lib.load()
    nbytes = lib.nntile_b200_tensor_flash_sdpa_scratch_bytes(_i64arr(shape5), _i64arr(base5))
    dev = tiled[0].tiles[0].device
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    keep = [t.pointers() for t in tiled]
    st = getattr(lib, name)(
        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), _i64arr(shape5),
        _i64arr(base5), *[ctypes.cast(p, ctypes.POINTER(ctypes.c_void_p)) for p in keep],
        ctypes.c_void_p(scratch.data_ptr()), nbytes)
    _lib.check(name, st)
    if scratch_holder is not None:
        scratch_holder.append(scratch)
    return scratch


def flash_sdpa_fwd_async(K, Q, mask, lse, V, A, seq_tile=None, batch_tile=None, scratch_out=None):
    """nntile.functions.flash_sdpa_fwd_cudnn_async on whole tensors: cuts them into
    tiles like the reference's traits do, runs the C tensor-level loops, gathers A
    and lse back in place.  Q, A: (H, G, B, S, D) bf16; K, V: the same shape, or
    (H, B, S, D) = [head, seq, batch, kv_heads] not replicated over the group
    (grouped-query form); mask: additive (Sq, Sk) bf16 buffer = Fortran [Sk, Sq];
    lse: (H, G, B, S) fp32."""
    H, G, B, S, D = Q.shape
    gqa = K.dim() == 4
    seq_tile = seq_tile or S
    bt = tuple(batch_tile or (B, G, H))
    base5 = (D, seq_tile) + bt
    kv_base = (D, seq_tile, bt[0], bt[2]) if gqa else base5
    tK, tV = TiledBuffer(K, kv_base), TiledBuffer(V, kv_base)
    tQ, tA = TiledBuffer(Q, base5), TiledBuffer(A, base5)
    tM = TiledBuffer(mask, (seq_tile, seq_tile))
    tL = TiledBuffer(lse, (seq_tile,) + bt)
    name = f"nntile_b200_tensor_flash_sdpa_fwd{'_gqa' if gqa else ''}_{ops._sfx16(Q)}"
    _tensor_call(name, (D, S, B, G, H), base5, [tK, tQ, tM, tL, tV, tA], scratch_out)
    A.copy_(tA.gather())
    lse.copy_(tL.gather())


def flash_sdpa_bwd_async(K, Q, V, A, dA, mask, lse, dK, dQ, dV, seq_tile=None,
                         batch_tile=None, scratch_out=None):
    """nntile.functions.flash_sdpa_bwd_cudnn_async on whole tensors (K, V, dK, dV
    5-D like Q, or 4-D un-replicated for the grouped-query form)."""
    H, G, B, S, D = Q.shape
    gqa = K.dim() == 4
    seq_tile = seq_tile or S
    bt = tuple(batch_tile or (B, G, H))
    base5 = (D, seq_tile) + bt
    kv_base = (D, seq_tile, bt[0], bt[2]) if gqa else base5
    tK, tV, tdK, tdV = (TiledBuffer(x, kv_base) for x in (K, V, dK, dV))
    tQ, tA, tdA, tdQ = (TiledBuffer(x, base5) for x in (Q, A, dA, dQ))
    tM = TiledBuffer(mask, (seq_tile, seq_tile))
    tL = TiledBuffer(lse, (seq_tile,) + bt)
    name = f"nntile_b200_tensor_flash_sdpa_bwd{'_gqa' if gqa else ''}_{ops._sfx16(Q)}"
    _tensor_call(name, (D, S, B, G, H), base5, [tK, tQ, tV, tA, tdA, tM, tL, tdK, tdQ, tdV],
                 scratch_out)
    dK.copy_(tdK.gather())
    dQ.copy_(tdQ.gather())
    dV.copy_(tdV.gather())


class _TiledChain:
    """Tile loops of the unfused chain: what nntile::tensor::gemm_async
    (src/tensor/gemm.cc:344-410: every output tile, contraction tiles accumulated
    with beta = 1 after the first), maxsumexp_async (src/tensor/maxsumexp.cc:80-107:
    the K tiles of a fibre accumulate into the same (max, sum) pair),
    softmax_inplace_async (src/tensor/softmax_inplace.cc:80-112), mask_scalar_async
    (src/tensor/mask_scalar.cc:26-62), sumprod_slice_async, add_slice_inplace_async
    and multiply_inplace_async do on tiled tensors, in the order
    nntile.layer.Sdpa issues them (sdpa.py:407-455, 595-698).  Tensors are cut along
    the sequence axis (queries and keys separately) and the three batch axes; the
    head axis is one tile."""

    def __init__(self, layer, q_tile, k_tile, batch_tile):
        self.L = layer
        H, G, B, Sq, D = layer.q.shape
        Sk = layer.k.shape[3]
        self.bt = tuple(batch_tile or (B, G, H))
        self.qt, self.kt = int(q_tile or Sq), int(k_tile or Sk)
        self.D, self.Sq, self.Sk = D, Sq, Sk
        self.nq, self.nk = -(-Sq//self.qt), -(-Sk//self.kt)
        self.nb = tuple(-(-s//t) for s, t in zip((B, G, H), self.bt))
        self.batch_tiles = self.nb[0]*self.nb[1]*self.nb[2]
        dev, dt = layer.q.device, layer.q.dtype
        self.attn_full = torch.empty((H, G, B, Sq, Sk), dtype=dt, device=dev)
        self.attn = TiledBuffer(self.attn_full, (self.kt, self.qt) + self.bt)
        self.mse = TiledBuffer(torch.empty((H, G, B, Sq, 2), dtype=dt, device=dev),
                               (2, self.qt) + self.bt)
        self.sps = TiledBuffer(torch.empty((H, G, B, Sq), dtype=dt, device=dev),
                               (self.qt,) + self.bt)
        self.mask = None if layer.mask is None else TiledBuffer(layer.mask, (self.kt, self.qt))

    def _cut(self, x, seq_tile):
        return TiledBuffer(x, (self.D, seq_tile) + self.bt)

    @staticmethod
    def _nbatch(t):
        return t.shape[0]*t.shape[1]*t.shape[2]

    def forward(self):
        L = self.L
        q, k, v = self._cut(L.q, self.qt), self._cut(L.k, self.kt), self._cut(L.v, self.kt)
        y = self._cut(L.y, self.qt)
        nq, nk = self.nq, self.nk
        for b in range(self.batch_tiles):
            for qi in range(nq):
                tq, ty, tm = q.tiles[qi + nq*b], y.tiles[qi + nq*b], self.mse.tiles[qi + nq*b]
                nbat, sq = self._nbatch(tq), tq.shape[3]
                ops.clear(tm)
                for ki in range(nk):
                    tk = k.tiles[ki + nk*b]
                    ta = self.attn.tiles[ki + nk*(qi + nq*b)]
                    sk = tk.shape[3]
                    ops.gemm(True, False, sk, sq, self.D, nbat, L.scale, tk, tq, 0.0, ta)
                    if self.mask is not None:
                        ops.mask_scalar(sk*sq, nbat, self.mask.tiles[ki + nk*qi], L.val, ta)
                    ops.maxsumexp(1, sq*nbat, sk, ta, tm)
                for ki in range(nk):
                    ta = self.attn.tiles[ki + nk*(qi + nq*b)]
                    sk = ta.shape[4]
                    ops.softmax_inplace(1, sq*nbat, sk, tm, 1.0, ta)
                    ops.gemm(False, False, self.D, sq, sk, nbat, 1.0, v.tiles[ki + nk*b], ta,
                             0.0 if ki == 0 else 1.0, ty)
        L.y.copy_(y.gather())
        L.attn = self.attn.gather()
        L.attn_maxsumexp = self.mse.gather()

    def backward(self, dy, dq, dk, dv):
        L = self.L
        q, k, v = self._cut(L.q, self.qt), self._cut(L.k, self.kt), self._cut(L.v, self.kt)
        y, tdy = self._cut(L.y, self.qt), self._cut(dy, self.qt)
        tdq, tdk, tdv = self._cut(dq, self.qt), self._cut(dk, self.kt), self._cut(dv, self.kt)
        nq, nk = self.nq, self.nk
        for b in range(self.batch_tiles):
            for qi in range(nq):
                tq, ty, tg = q.tiles[qi + nq*b], y.tiles[qi + nq*b], tdy.tiles[qi + nq*b]
                tsp = self.sps.tiles[qi + nq*b]
                nbat, sq = self._nbatch(tq), tq.shape[3]
                ops.sumprod_slice(1, sq*nbat, self.D, 1.0, ty, tg, 0.0, tsp)
                for ki in range(nk):
                    tk, tv = k.tiles[ki + nk*b], v.tiles[ki + nk*b]
                    ta = self.attn.tiles[ki + nk*(qi + nq*b)]
                    sk = tk.shape[3]
                    da = torch.empty_like(ta)
                    ops.gemm(True, False, sk, sq, self.D, nbat, 1.0, tv, tg, 0.0, da)
                    ops.gemm(False, True, self.D, sk, sq, nbat, 1.0, tg, ta, 1.0,
                             tdv.tiles[ki + nk*b])
                    ops.add_slice_inplace(1, sq*nbat, sk, -1.0, tsp, 1.0, da)
                    ops.multiply_inplace(da.numel(), 1.0, ta, da)
                    if self.mask is not None:
                        ops.mask_scalar(sk*sq, nbat, self.mask.tiles[ki + nk*qi], 0.0, da)
                    ops.gemm(False, True, self.D, sk, sq, nbat, L.scale, tq, da, 1.0,
                             tdk.tiles[ki + nk*b])
                    ops.gemm(False, False, self.D, sq, sk, nbat, L.scale, tk, da, 1.0,
                             tdq.tiles[qi + nq*b])
        dq.copy_(tdq.gather())
        dk.copy_(tdk.gather())
        dv.copy_(tdv.gather())


class Sdpa:
    """Mirror of nntile.layer.Sdpa on tensors that are one tile or are cut along
    the sequence and batch axes (``seq_tile`` for queries and keys alike, or
    ``q_tile`` / ``k_tile`` separately for the unfused chain; ``batch_tile`` =
    (batch, group, kv_heads) extents of a tile).

    q, k, v: (H, G, B, S, D) buffers; for the fused path k and v may also be
    (H, B, S, D), not replicated over the group (grouped-query form).  ``mask``:
    for the unfused chain a bool (Sq, Sk) buffer = Fortran [Sk, Sq] (true = keep);
    for the fused path the additive mask in the tensors' dtype (0 / -inf), as
    sdpa.py:457-531 prepares.
    """

    def __init__(self, q, k, v, mask=None, flash_attention=False, seq_tile=None,
                 batch_tile=None, q_tile=None, k_tile=None):
        self.q, self.k, self.v, self.mask = q, k, v, mask
        self.flash_attention = flash_attention
        self.seq_tile, self.batch_tile = seq_tile, batch_tile
        self.q_tile, self.k_tile = q_tile or seq_tile, k_tile or seq_tile
        H, G, B, S, D = q.shape
        self.head, self.n_seq = D, S
        self.n_seq_k = k.shape[-2]
        self.batch = H*G*B
        self.scale = sdpa_scale(D)
        self.val = -math.inf
        dev, dt = q.device, q.dtype
        self.y = torch.zeros_like(q)
        if flash_attention:
            if dt not in (torch.bfloat16, torch.float16):
                raise TypeError("the fused path takes bf16 or fp16 (fp32 is rejected by the "
                                "reference as well, flash_sdpa_fwd_cudnn/cuda.cc:60-63)")
            self.flash_logsumexp = torch.empty((H, G, B, S), dtype=torch.float32, device=dev)
            if mask is None:
                self.mask = torch.zeros((S, S), dtype=dt, device=dev)
        elif self._tiled():
            self._chain = _TiledChain(self, self.q_tile, self.k_tile, batch_tile)
        else:
            self.attn = torch.empty((H, G, B, S, self.n_seq_k), dtype=dt, device=dev)
            self.attn_maxsumexp = torch.empty((H, G, B, S, 2), dtype=dt, device=dev)
            self.attn_sumprod_slice = torch.empty((H, G, B, S), dtype=dt, device=dev)

    def _tiled(self) -> bool:
        H, G, B, S, D = self.q.shape
        return bool((self.q_tile and self.q_tile < S)
                    or (self.k_tile and self.k_tile < self.n_seq_k)
                    or (self.batch_tile and tuple(self.batch_tile) != (B, G, H)))

    # ---- forward ----------------------------------------------------------
    def forward_async(self):
        if self.flash_attention:
            ops.fill(-math.inf, self.flash_logsumexp)          # sdpa.py:538
            ops.clear(self.y)                                   # sdpa.py:539
            flash_sdpa_fwd_async(self.k, self.q, self.mask, self.flash_logsumexp, self.v,
                                 self.y, self.seq_tile, self.batch_tile)
            return self.y
        if self._tiled():
            self._chain.forward()
            return self.y
        D, Sq, Sk, nb = self.head, self.n_seq, self.n_seq_k, self.batch
        ops.gemm(True, False, Sk, Sq, D, nb, self.scale, self.k, self.q, 0.0, self.attn)
        ops.clear(self.attn_maxsumexp)
        if self.mask is not None:
            ops.mask_scalar(Sk*Sq, nb, self.mask, self.val, self.attn)
        ops.maxsumexp(1, Sq*nb, Sk, self.attn, self.attn_maxsumexp)
        ops.softmax_inplace(1, Sq*nb, Sk, self.attn_maxsumexp, 1.0, self.attn)
        ops.gemm(False, False, D, Sq, Sk, nb, 1.0, self.v, self.attn, 0.0, self.y)
        return self.y

    def forward_dynamic(self, q, k, v, mask=None, kv_cache=None):
        """nntile.layer.Sdpa.forward_dynamic (sdpa.py:170-306): forward on tensors
        handed in at call time - the key/value sequence may be longer than the query
        sequence (generation against a cache) - with temporaries allocated on the
        fly; no backward.  As there, the fused path runs only when the two sequence
        lengths agree; otherwise the unfused chain.  ``mask`` is what the
        constructor takes for the chosen path.

        Beyond the reference: with ``kv_cache`` (a KVCache or PagedKVCache holding the
        un-replicated keys and values) and a single query position, the split-KV decode
        kernel reads the filled part of the cache in place; k and v are then ignored."""
        H, G, B, Sq, D = q.shape
        if kv_cache is not None and Sq == 1 and len(kv_cache) > 0:
            return kv_cache.decode(q)
        Sk = k.shape[3]
        mask_local = mask if mask is not None else self.mask
        y = torch.zeros_like(q)
        nb = H*G*B
        if self.flash_attention and Sk == Sq:
            lse = torch.full((H, G, B, Sq), -math.inf, dtype=torch.float32, device=q.device)
            if mask_local is None:
                mask_local = torch.zeros((Sq, Sq), dtype=q.dtype, device=q.device)
            flash_sdpa_fwd_async(k, q, mask_local, lse, v, y, self.seq_tile, self.batch_tile)
            return y
        attn = torch.empty((H, G, B, Sq, Sk), dtype=q.dtype, device=q.device)
        attn_max = torch.zeros((H, G, B, Sq, 2), dtype=q.dtype, device=q.device)
        ops.gemm(True, False, Sk, Sq, D, nb, sdpa_scale(D), k, q, 0.0, attn)
        if mask_local is not None:
            ops.mask_scalar(Sk*Sq, nb, mask_local, self.val, attn)
        ops.maxsumexp(1, Sq*nb, Sk, attn, attn_max)
        ops.softmax_inplace(1, Sq*nb, Sk, attn_max, 1.0, attn)
        ops.gemm(False, False, D, Sq, Sk, nb, 1.0, v, attn, 0.0, y)
        return y

    # ---- backward: dq, dk, dv are INCREMENTED, as in the reference -----------
    def backward_async(self, dy, dq, dk, dv):
        if self.flash_attention:
            flash_sdpa_bwd_async(self.k, self.q, self.v, self.y, dy, self.mask,
                                 self.flash_logsumexp, dk, dq, dv, self.seq_tile,
                                 self.batch_tile)
            return
        if self._tiled():
            self._chain.backward(dy, dq, dk, dv)
            return
        D, Sq, Sk, nb = self.head, self.n_seq, self.n_seq_k, self.batch
        dattn = torch.empty_like(self.attn)
        ops.gemm(True, False, Sk, Sq, D, nb, 1.0, self.v, dy, 0.0, dattn)
        ops.gemm(False, True, D, Sk, Sq, nb, 1.0, dy, self.attn, 1.0, dv)
        ops.sumprod_slice(1, Sq*nb, D, 1.0, self.y, dy, 0.0, self.attn_sumprod_slice)
        ops.add_slice_inplace(1, Sq*nb, Sk, -1.0, self.attn_sumprod_slice, 1.0, dattn)
        ops.multiply_inplace(dattn.numel(), 1.0, self.attn, dattn)
        if self.mask is not None:
            ops.mask_scalar(Sk*Sq, nb, self.mask, 0.0, dattn)
        ops.gemm(False, True, D, Sk, Sq, nb, self.scale, self.q, dattn, 1.0, dk)
        ops.gemm(False, False, D, Sq, Sk, nb, self.scale, self.k, dattn, 1.0, dq)


def decode_sdpa(q, Kcache, Vcache, length=None, out=None, lse_out=None, workspace=None):
    """One new token against the cache.  q: (H, G, B, 1, D) bf16; caches:
    (H, B, L, D) bf16 = Fortran [D, L, B, H].  Returns out shaped like q."""
    H, G, B, one, D = q.shape
    L = Kcache.shape[2]
    length = L if length is None else int(length)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        n = ops.decode_workspace_bytes(D, length, B, G, H)
        workspace = torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)
    ops.decode_sdpa(D, L, length, B, G, H, q, Kcache, Vcache, out, lse_out, workspace)
    return out


class KVCache:
    """Preallocated key/value cache of one attention layer, filled in place.

    Mirrors nntile.layer.cache_utils.KVCache (wrappers/python/nntile/layer/
    cache_utils.py:118-228): ``append(k_partial, v_partial)``, ``len()``,
    ``clear()``, attributes ``k`` and ``v``.  Differences, all on purpose: the
    buffers hold the kv heads only (the reference stores what the attention layer
    has already replicated ``group`` times), ``append`` writes into the buffer at
    the current length (one kernel, no re-allocation), and there is no
    ``k_partial`` / ``v_partial`` copy of the filled part per step: ``decode``
    hands the whole buffer and the current length to the split-KV kernel.

    Torch shapes: k, v (kv_heads, batch, max_seq, head) = Fortran
    [head, max_seq, batch, kv_heads]; k_partial, v_partial (kv_heads, batch, new_seq,
    head); q (kv_heads, group, batch, 1, head)."""

    def __init__(self, max_cache_size: int, kv_heads: int, batch: int, head: int,
                 device="cuda"):
        self.max_cache_size = int(max_cache_size)
        self.k = torch.zeros((kv_heads, batch, self.max_cache_size, head), dtype=torch.bfloat16,
                             device=device)
        self.v = torch.zeros_like(self.k)
        self.k_cache_size = 0
        self.v_cache_size = 0
        self._workspace = None

    def append(self, k_partial: torch.Tensor, v_partial: torch.Tensor):
        H, B, L, D = self.k.shape
        if k_partial.shape != v_partial.shape or k_partial.shape[:2] != (H, B) \
                or k_partial.shape[3] != D:
            raise ValueError("k_partial / v_partial do not match the cache")
        n = k_partial.shape[2]
        ops.kv_cache_append(D, L, B, H, self.k_cache_size, n, k_partial.contiguous(), self.k)
        ops.kv_cache_append(D, L, B, H, self.v_cache_size, n, v_partial.contiguous(), self.v)
        self.k_cache_size += n
        self.v_cache_size += n

    def decode(self, q: torch.Tensor, out=None, lse_out=None):
        """Attention of one new query token per (batch, head) over the filled part."""
        H, G, B, one, D = q.shape
        need = ops.decode_workspace_bytes(D, max(self.k_cache_size, 1), B, G, H)
        if self._workspace is None or self._workspace.numel() < need:
            self._workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
        return decode_sdpa(q, self.k, self.v, length=self.k_cache_size, out=out,
                           lse_out=lse_out, workspace=self._workspace)

    def clear(self):
        self.k_cache_size = 0
        self.v_cache_size = 0

    def __len__(self):
        return self.k_cache_size


_ROWS = (torch.bfloat16, torch.float16)


class KVPages:
    """Buffers of a paged cache: what the paged_* functions read and write.

    Torch shapes: k, v (num_pages, kv_heads, page_size, head), bfloat16 or float16, or 8-bit
    e4m3 codes (uint8 or float8_e4m3fn) with k_scales, v_scales uint8 (num_pages, kv_heads,
    page_size), value = code * 2**(byte - 127); bounds, for paged_select, (num_pages,
    kv_heads, 2, head) in the type of the rows: least and largest stored key of a page."""

    __slots__ = ("k", "v", "k_scales", "v_scales", "bounds", "e4m3")

    def __init__(self, k, v, k_scales=None, v_scales=None, bounds=None):
        shape, dtype = k.shape, k.dtype
        if len(shape) != 4 or shape != v.shape or dtype != v.dtype:
            raise ValueError("k and v pages must be two equal (num_pages, kv_heads, page_size, "
                             "head) buffers")
        self.e4m3 = dtype not in _ROWS
        if self.e4m3:
            if dtype not in (torch.uint8, torch.float8_e4m3fn):
                raise TypeError(f"pages hold bfloat16, float16 or 8-bit codes, not {dtype}")
            for s in (k_scales, v_scales):
                if s is None or s.shape != shape[:3] or s.dtype != torch.uint8:
                    raise ValueError("8-bit pages need uint8 scales (num_pages, kv_heads, "
                                     "page_size) for k and v")
        elif k_scales is not None or v_scales is not None:
            raise ValueError("only 8-bit pages have scales")
        if bounds is not None and (bounds.shape != (shape[0], shape[1], 2, shape[3])
                                   or (not self.e4m3 and bounds.dtype != dtype)):
            raise ValueError("bounds must be (num_pages, kv_heads, 2, head) in the type of the rows")
        self.k, self.v, self.k_scales, self.v_scales, self.bounds = k, v, k_scales, v_scales, bounds

    @classmethod
    def empty(cls, num_pages, page_size, kv_heads, head, dtype=torch.bfloat16, e4m3=False,
              bounds=False, device="cuda"):
        shape = (num_pages, kv_heads, page_size, head)
        k, v = (torch.zeros(shape, dtype=torch.uint8 if e4m3 else dtype, device=device)
                for _ in range(2))
        ks, vs = ((torch.full(shape[:3], 127, dtype=torch.uint8, device=device)
                   for _ in range(2)) if e4m3 else (None, None))
        bd = torch.zeros((num_pages, kv_heads, 2, head), dtype=dtype, device=device) \
            if bounds else None
        return cls(k, v, ks, vs, bd)

    def _check_rows(self, t, what):
        dtype = t.dtype
        if dtype not in _ROWS or (not self.e4m3 and dtype != self.k.dtype):
            raise TypeError(f"{what} is {dtype}, the pages hold {self.k.dtype}")


def _check_table(lengths, block_table, batch):
    """max_blocks of a table that fits."""
    if lengths.dtype != torch.int32 or block_table.dtype != torch.int32:
        raise TypeError("lengths and block_table must be int32")
    shape = block_table.shape
    if lengths.shape != (batch,) or len(shape) != 2 or shape[0] != batch:
        raise ValueError("lengths must be (batch,) and block_table (batch, max_blocks)")
    return shape[1]


def _check_status(status):
    if status is not None and (status.dtype not in (torch.int32, torch.uint32)
                               or status.numel() != 1):
        raise ValueError("status must be one 32-bit word")


def paged_append(pages, lengths, block_table, k, v, new_lens=None, status=None):
    """Write rows k, v (kv_heads, batch, new_seq, head) behind the lengths[b] filled positions
    of every sequence (the first new_lens[b] of them; default all).  Changes the pages, their
    scales and bounds, not `lengths` and `block_table`.  `status`: optional 32-bit word that
    receives NNTILE_B200_PAGED_BAD_* bits."""
    if _paged_torch is not None:
        done = _paged_torch.append(pages, lengths, block_table, k, v, new_lens, status)
        if done is True:
            return
    N, H, P, D = pages.k.shape
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[0] != H or shape[3] != D:
        raise ValueError("k and v must be (kv_heads, batch, new_seq, head) rows for these pages")
    pages._check_rows(k, "k")
    if v.dtype != k.dtype or (pages.bounds is not None and pages.bounds.dtype != k.dtype):
        raise TypeError("k, v and the bounds must have one type")
    B, n = shape[1], shape[2]
    M = _check_table(lengths, block_table, B)
    if new_lens is not None and (new_lens.dtype != torch.int32 or new_lens.shape != (B,)):
        raise ValueError("new_lens must be int32 (batch,)")
    _check_status(status)
    ops.paged_kv_append(D, P, N, M, B, H, n, int(pages.e4m3), lengths, new_lens,
                        block_table, k, v, pages.k, pages.v, pages.k_scales, pages.v_scales,
                        pages.bounds, status)


def paged_gather(pages, lengths, block_table, k, v, status=None):
    """Read the cache into k, v (kv_heads, batch, max_seq, head): rows 0 .. lengths[b] - 1 of
    every sequence; rows behind them are left as they are."""
    if _paged_torch is not None:
        done = _paged_torch.gather(pages, lengths, block_table, k, v, status)
        if done is True:
            return
    N, H, P, D = pages.k.shape
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[0] != H or shape[3] != D:
        raise ValueError("k and v must be (kv_heads, batch, max_seq, head) buffers for these pages")
    pages._check_rows(k, "k")
    if v.dtype != k.dtype:
        raise TypeError("k and v must have one type")
    B = shape[1]
    M = _check_table(lengths, block_table, B)
    _check_status(status)
    ops.paged_kv_gather(D, P, N, M, B, H, shape[2], int(pages.e4m3), lengths,
                        block_table, pages.k, pages.v, pages.k_scales, pages.v_scales, k, v,
                        status)


def _check_query(q, pages):
    """(num_pages, kv_heads, page_size, head, group, batch) of a query that fits."""
    N, H, P, D = pages.k.shape
    shape = q.shape
    if len(shape) != 5 or shape[0] != H or shape[3] != 1 or shape[4] != D:
        raise ValueError("q must be (kv_heads, group, batch, 1, head) for these pages")
    pages._check_rows(q, "q")
    return N, H, P, D, shape[1], shape[2]


def paged_select(q, pages, lengths, block_table, num_selected, first_blocks=1, last_blocks=1,
                 out=None, workspace=None, status=None):
    """Blocks that the new token of every sequence attends to, per kv head: the first and the
    last ones and those whose bounds allow the highest score.  Returns int32 (kv_heads,
    batch, num_selected), ascending block numbers, then -1."""
    if _paged_torch is not None:
        done = _paged_torch.select(q, pages, lengths, block_table, num_selected, first_blocks,
                                   last_blocks, out, workspace, status)
        if isinstance(done, torch.Tensor):
            return done
    N, H, P, D, G, B = _check_query(q, pages)
    if pages.bounds is None:
        raise ValueError("these pages keep no bounds")
    if pages.bounds.dtype != q.dtype:
        raise TypeError("q and the bounds must have one type")
    M = _check_table(lengths, block_table, B)
    _check_status(status)
    if out is None:
        out = torch.empty((H, B, num_selected), dtype=torch.int32, device=q.device)
        if G == 0:                              # no query, nothing selected: the call writes nothing
            out.fill_(-1)
    elif out.shape != (H, B, num_selected) or out.dtype != torch.int32:
        raise ValueError("out must be int32 (kv_heads, batch, num_selected)")
    if workspace is None:
        need = ops.paged_select_workspace_bytes(M, B, H)
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    ops.paged_select(D, P, N, M, B, G, H, num_selected, first_blocks, last_blocks, lengths,
                     block_table, q, pages.bounds, out, workspace, status)
    return out


def paged_decode(q, pages, lengths, block_table, selected=None, out=None, lse_out=None,
                 workspace=None, status=None):
    """decode_sdpa over a paged cache: one new token q (kv_heads, group, batch, 1, head) per
    sequence against its first lengths[b] positions, or against those of them in the blocks
    of `selected` (int32 (kv_heads, batch, num_selected), as paged_select returns).  Returns
    out shaped like q; lse_out: optional float32 (kv_heads, group, batch)."""
    if _paged_torch is not None:
        done = _paged_torch.decode(q, pages, lengths, block_table, selected, out, lse_out,
                                   workspace, status)
        if isinstance(done, torch.Tensor):
            return done
    N, H, P, D, G, B = _check_query(q, pages)
    M, S = _check_table(lengths, block_table, B), 0
    _check_status(status)
    if selected is not None:
        shape = selected.shape
        if selected.dtype != torch.int32 or len(shape) != 3 or shape[:2] != (H, B) or shape[2] == 0:
            raise ValueError("selected must be int32 (kv_heads, batch, num_selected)")
        S = shape[2]
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must be like q")
    if lse_out is not None and (lse_out.dtype != torch.float32 or lse_out.numel() != H*G*B):
        raise ValueError("lse_out must be float32 (kv_heads, group, batch)")
    if workspace is None:
        need = ops.paged_decode_workspace_bytes(D, P, M, B, G, H, S)
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    ops.paged_decode_sdpa(D, P, N, M, B, G, H, S, int(pages.e4m3), lengths, block_table, selected,
                          q, pages.k, pages.v, pages.k_scales, pages.v_scales, out, lse_out,
                          workspace, status)
    return out


class PagedKVCache:
    """Key/value cache of one attention layer in a pool of pages; sequences grow, and are
    released, independently of one another.

    The paged counterpart of KVCache, with the same `append`, `decode`, `clear` and `len()`
    (the longest sequence), so `Sdpa.forward_dynamic` takes either.  Pages are handed out and
    taken back on the host; tables and lengths are kept on the device.  `e4m3` halves the
    cache; `bounds` keeps what `decode(..., num_selected=...)` needs to attend to selected
    blocks only.  For a captured graph call paged_append / paged_select / paged_decode on
    `pages`, `lengths` and `block_table`: append() here does host bookkeeping."""

    def __init__(self, num_pages, page_size, kv_heads, batch, head, max_blocks=None,
                 dtype=torch.bfloat16, e4m3=False, bounds=False, device="cuda"):
        self.pages = KVPages.empty(num_pages, page_size, kv_heads, head, dtype, e4m3, bounds,
                                   device)
        self.dtype, self.page_size = dtype, int(page_size)
        self.max_blocks = int(num_pages if max_blocks is None else max_blocks)
        self.block_table = torch.full((batch, self.max_blocks), -1, dtype=torch.int32,
                                      device=device)
        self.lengths = torch.zeros((batch,), dtype=torch.int32, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._tables = [[] for _ in range(batch)]
        self._filled = [0]*batch

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequence_lengths(self) -> list[int]:
        return list(self._filled)

    def append(self, k_partial, v_partial, new_lens=None):
        """Rows (kv_heads, batch, new_seq, head); new_lens: how many of them count for every
        sequence (a list of ints; default all).  Raises, with nothing changed, when the pool
        or a sequence's table has no room."""
        batch = len(self._filled)
        if k_partial.dim() != 4 or k_partial.shape != v_partial.shape \
                or k_partial.shape[1] != batch:
            raise ValueError("k_partial / v_partial do not match the cache")
        self.pages._check_rows(k_partial, "k_partial")
        if k_partial.dtype != self.dtype:
            raise TypeError(f"rows are {k_partial.dtype}, the cache keeps {self.dtype}")
        n = k_partial.shape[2]
        new = [n]*batch if new_lens is None else [int(x) for x in new_lens]
        if len(new) != batch or any(x < 0 or x > n for x in new):
            raise ValueError("new_lens must be batch numbers between 0 and new_seq")
        P = self.page_size
        more = [-(-(f + x)//P) - len(t) for f, x, t in zip(self._filled, new, self._tables)]
        if any(len(t) + m > self.max_blocks for t, m in zip(self._tables, more)):
            raise ValueError("a sequence would pass max_blocks pages")
        if sum(more) > len(self._free):
            raise ValueError(f"the pool has {len(self._free)} free pages, {sum(more)} are needed")
        device = self.lengths.device
        left = len(self._free) - sum(more)
        pages, entries = iter(self._free[:left - 1 if left else None:-1]), []
        for b, m in enumerate(more):
            entries += [(b, len(self._tables[b]) + i, next(pages)) for i in range(m)]
        if entries:
            rows = torch.tensor(entries, dtype=torch.int64).to(device)
            self.block_table[rows[:, 0], rows[:, 1]] = rows[:, 2].to(torch.int32)
        lens = None if new_lens is None else torch.tensor(new, dtype=torch.int32).to(device)
        paged_append(self.pages, self.lengths, self.block_table, k_partial.contiguous(),
                     v_partial.contiguous(), lens)
        # the rows are on their way: from here on the pages are taken (until then only table
        # entries behind the lengths have changed, which nothing reads)
        self.lengths += n if lens is None else lens
        del self._free[left:]
        for b, _, page in entries:
            self._tables[b].append(page)
        self._filled = [f + x for f, x in zip(self._filled, new)]

    def decode(self, q, out=None, lse_out=None, num_selected=None, first_blocks=1, last_blocks=1):
        """Attention of one new token per sequence over everything that is filled, or over
        num_selected blocks per kv head."""
        selected = None
        if num_selected is not None:
            selected = paged_select(q, self.pages, self.lengths, self.block_table, num_selected,
                                    first_blocks, last_blocks)
        return paged_decode(q, self.pages, self.lengths, self.block_table, selected, out, lse_out)

    def read(self):
        """The filled part as contiguous k, v (kv_heads, batch, len(self), head); zeros behind
        shorter sequences."""
        N, H, P, D = self.pages.k.shape
        k = torch.zeros((H, len(self._filled), len(self), D), dtype=self.dtype,
                        device=self.lengths.device)
        v = torch.zeros_like(k)
        paged_gather(self.pages, self.lengths, self.block_table, k, v)
        return k, v

    def release(self, b: int):
        """Sequence b ends: its pages go back to the pool, its slot is empty."""
        self._free.extend(reversed(self._tables[b]))
        self._tables[b] = []
        self._filled[b] = 0
        self.lengths[b] = 0
        self.block_table[b] = -1

    def clear(self):
        for b in range(len(self._filled)):
            self.release(b)

    def __len__(self):
        return max(self._filled, default=0)
