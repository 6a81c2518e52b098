"""Pages of a 4-bit latent cache that many sequences share, and the decode attention over them.

The reference decodes one sequence over one contiguous cache (kernel/palu_attention.py:207-257); a server holds many sequences
that grow, share a prompt and end.  Here the packed latents of all of them live in one pool of pages:

    pool.k_codes uint8 [N, G, P, Rk / 2]   pool.k_meta fp16 [N, G, P, 2] = (scale, zero)   pool.v_codes / pool.v_meta alike

(`palu_amd.kernel.quant.quantize_pack` rows with 4 bits), with a leading axis of layers where one allocation serves a whole model.
Row b of an int32 block table lists the pages of sequence b; position l of the sequence is row l % P of its page l // P.

  `paged_append`  quantises rows of any mix of sequences straight into their pages
  `paged_copy`    copies whole pages in all layers (a fork's open page, compaction)
  `paged_attn`    one new token of each of B sequences against its pages
  `PagedLatentCache`  the pool with its bookkeeping: sequences, reference counts, fork / free / compact

Everything runs on the current stream and allocates only through torch's caching allocator (graph-capturable).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib
from .abx_rope import rope_inv_freq

__all__ = ["PagePool", "make_pool", "paged_append", "paged_attn", "paged_copy", "prepare_paged_b"]


class PagePool(tuple):
    """The four arrays of a pool (k_codes, k_meta, v_codes, v_meta): contiguous, on one GPU, [N, G, P, ...] or [layers, N, G, P, ...].
    Checked once, when it is made; a program keeps it as it keeps the arrays.  num_pages, num_groups, page_size, rank_k, rank_v (ranks
    of one group) and layers (1 without the axis) are its sizes."""

    def __new__(cls, k_codes: torch.Tensor, k_meta: torch.Tensor, v_codes: torch.Tensor, v_meta: torch.Tensor):
        arrays = (k_codes, k_meta, v_codes, v_meta)
        if k_codes.dim() not in (4, 5):
            raise ValueError(f"PagePool: the arrays must be [layers,] [N, G, P, ...], got {tuple(k_codes.shape)}")
        lead, dev = k_codes.shape[:-1], k_codes.device
        if v_codes.shape[:-1] != lead or k_meta.shape != (*lead, 2) or v_meta.shape != (*lead, 2):
            raise ValueError(f"PagePool: the arrays disagree: {[tuple(t.shape) for t in arrays]}")
        if any(t.dtype != d for t, d in zip(arrays, (torch.uint8, torch.float16) * 2)):
            raise TypeError(f"PagePool: codes are uint8 and meta fp16, got {[t.dtype for t in arrays]}")
        if any(t.device != dev for t in arrays):
            raise ValueError(f"PagePool: the arrays must lie on one device, got {[str(t.device) for t in arrays]}")
        if not all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in arrays):
            raise ValueError("PagePool: the arrays must be contiguous and 16-byte aligned")
        self = super().__new__(cls, arrays)
        self.layered = k_codes.dim() == 5
        self.layers = lead[0] if self.layered else 1
        self.num_pages, self.num_groups, self.page_size = lead[-3:]
        self.rank_k, self.rank_v = 2 * k_codes.shape[-1], 2 * v_codes.shape[-1]
        self.device = dev
        if min(lead) < 1:
            raise ValueError("PagePool: the pool is empty")
        if self.page_size < 16 or self.page_size & (self.page_size - 1):
            raise ValueError(f"PagePool: the page size must be a power of two >= 16, got {self.page_size}")
        if any(r % 8 or r < 8 or r > 512 for r in (self.rank_k, self.rank_v)):
            raise ValueError(f"PagePool: group ranks must be multiples of 8 up to 512, got {self.rank_k}, {self.rank_v}")
        self._ptrs = tuple(t.data_ptr() for t in arrays)
        return self

    k_codes = property(lambda self: self[0])
    k_meta = property(lambda self: self[1])
    v_codes = property(lambda self: self[2])
    v_meta = property(lambda self: self[3])

    def layer(self, i: int) -> "PagePool":
        """The pool of layer i of a pool with an axis of layers (views)."""
        if not self.layered:
            raise ValueError("PagePool.layer: this pool has no axis of layers")
        return PagePool(*(t[i] for t in self))


def make_pool(num_pages: int, num_groups: int, page_size: int, rank_k: int, rank_v: int, layers: Optional[int] = None,
              device="cuda") -> PagePool:
    """An empty pool (rank_k / rank_v: ranks of ONE group).  Rows are zero until written."""
    lead = (num_pages,) if layers is None else (layers, num_pages)

    def t(last, dtype):
        return torch.zeros((*lead, num_groups, page_size, last), dtype=dtype, device=device)
    return PagePool(t(rank_k // 2, torch.uint8), t(2, torch.float16), t(rank_v // 2, torch.uint8), t(2, torch.float16))


def _pool(pool: PagePool, what: str, layers: bool = False) -> PagePool:
    if type(pool) is not PagePool:
        raise TypeError(f"{what}: the pool must be a PagePool")
    if not pool[0].is_cuda:
        raise TypeError(f"{what}: the pool must lie on a ROCm device (no CPU fallback)")
    if pool.layered and not layers:
        raise ValueError(f"{what}: one layer at a time (pick a layer: pool.layer(i))")
    return pool


def _launch(dev, fn, name: str, *args):
    """fn(*args, stream) on the current stream of `dev`, which is made the current device if it is not"""
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, _lib.current_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.current_stream(dev))
    if rc:
        _lib.check(rc, name)


def _int32(t: torch.Tensor, name: str, dim: int, dev, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim:
        raise TypeError(f"{what}: {name} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''}")
    if t.device != dev:
        raise ValueError(f"{what}: {name} must lie on {dev}, it is on {t.device}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def paged_append(pool: PagePool, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_ids: torch.Tensor,
                 positions: torch.Tensor) -> None:
    """Quantise the latent rows k [T, G, Rk], v [T, G, Rv] (fp16) to 4 bits and write row t as position positions[t] of sequence
    seq_ids[t] of `block_table` [B, max_pages]: the codes and (scale, zero) pairs are bit for bit those of `quantize_pack`.

    The rows may come in any order and belong to any mix of sequences (one decode token each, whole prompts).  A negative id or
    position marks a padding row and is skipped, like a row whose sequence, table entry or page does not exist.  No two rows of a
    call may name the same place."""
    what = "paged_append"
    _pool(pool, what)
    dev, G, Rk, Rv = pool.device, pool.num_groups, pool.rank_k, pool.rank_v
    for t, name, R in ((k, "k", Rk), (v, "v", Rv)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.device != dev:
            raise TypeError(f"{what}: {name} must be an fp16 tensor on the pool's device")
        if t.dim() != 3 or t.shape[1] != G or t.shape[2] != R:
            raise ValueError(f"{what}: {name} must be [T, {G}, {R}], got {tuple(t.shape)}")
    T = k.shape[0]
    table = _int32(block_table, "block_table", 2, dev, what)
    seq, pos = _int32(seq_ids, "seq_ids", 1, dev, what), _int32(positions, "positions", 1, dev, what)
    if v.shape[0] != T or seq.shape[0] != T or pos.shape[0] != T:
        raise ValueError(f"{what}: k, v, seq_ids and positions must have one entry per row ({T})")
    B, M = table.shape
    if T == 0 or B == 0 or M == 0:
        return
    k, v = _rows16(k), _rows16(v)
    _launch(dev, _lib.lib.palu_paged_append_q4, "palu_paged_append_q4", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), *pool._ptrs, table.data_ptr(), table.stride(0), B, M, seq.data_ptr(), pos.data_ptr(), T, G,
            pool.page_size, pool.num_pages, Rk, Rv)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """rows the kernels can load 16 bytes at a time"""
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _page_pairs(pages, name: str, n_pages: int, dev, what: str):
    """a list (checked here) or an int32 tensor on the device -> (device tensor, list or None)"""
    if isinstance(pages, torch.Tensor) and pages.is_cuda:
        t = _int32(pages, name, 1, dev, what)
        return (t if t.is_contiguous() else t.contiguous()), None
    lst = pages.tolist() if isinstance(pages, torch.Tensor) else list(pages)
    for i in lst:
        if not isinstance(i, int) or not 0 <= i < n_pages:
            raise ValueError(f"{what}: {name} names page {i!r}, the pool has pages 0 .. {n_pages - 1}")
    return None, lst


def paged_copy(pool: PagePool, src, dst) -> None:
    """Page dst[i] becomes a copy of page src[i], in every layer of the pool, in one launch.

    `src` and `dst`: sequences of ints (checked: pages of the pool, targets distinct and no source among them), or int32 tensors on
    the pool's device, for which the caller answers for that (a pair that names no page of the pool is skipped)."""
    what = "paged_copy"
    _pool(pool, what, layers=True)
    dev, N = pool.device, pool.num_pages
    s, s_list = _page_pairs(src, "src", N, dev, what)
    d, d_list = _page_pairs(dst, "dst", N, dev, what)
    if (s_list is None) != (d_list is None):
        raise TypeError(f"{what}: src and dst must both be tensors on the device, or both be on the host")
    if s_list is not None:
        if len(s_list) != len(d_list):
            raise ValueError(f"{what}: {len(s_list)} sources for {len(d_list)} targets")
        if len(set(d_list)) != len(d_list) or set(d_list) & set(s_list):
            raise ValueError(f"{what}: the targets must be distinct and none of them a source")
        if not s_list:
            return
        s, d = torch.tensor([s_list, d_list], dtype=torch.int32).to(dev)
    elif s.shape != d.shape:
        raise ValueError(f"{what}: {s.shape[0]} sources for {d.shape[0]} targets")
    n = s.shape[0]
    if n == 0:
        return
    _launch(dev, _lib.lib.palu_paged_copy, "palu_paged_copy", *pool._ptrs, s.data_ptr(), d.data_ptr(), n, pool.layers, N,
            pool.num_groups, pool.page_size, pool.rank_k, pool.rank_v)


def prepare_paged_b(b: torch.Tensor, num_groups: int) -> torch.Tensor:
    """The key reconstruction B [H, Rk, 128] fp16 (`HeadwiseLowRankModule.B`, kernel/palu_attention.py:108-114) in the layout that
    `paged_attn` reads: a weight, laid out once."""
    if not b.is_cuda or b.dtype != torch.float16 or b.dim() != 3:
        raise TypeError("prepare_paged_b: B must be an fp16 ROCm tensor [H, Rk, 128] (no CPU fallback)")
    H, Rk, D = b.shape
    n = _lib.lib.palu_paged_b_bytes(H, num_groups, Rk)
    if n == 0 or D != 128:
        raise ValueError(f"prepare_paged_b: need H % num_groups == 0, head_dim 128 and a group rank that is a multiple of 8 up to "
                         f"256; got H={H}, num_groups={num_groups}, Rk={Rk}, head_dim={D}")
    b = b.contiguous()
    out = torch.empty(n, dtype=torch.uint8, device=b.device)
    _launch(b.device, _lib.lib.palu_paged_prepare_b, "palu_paged_prepare_b", b.data_ptr(), H, num_groups, Rk, D, out.data_ptr())
    return out


def paged_attn(q: torch.Tensor, bfrag: torch.Tensor, pool: PagePool, block_table: torch.Tensor, seq_lens: torch.Tensor,
               q_positions: Optional[torch.Tensor] = None, theta: float = 10000.0, sm_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token of each of B sequences over its cached latents (the decode branch, kernel/palu_attention.py:
    207-251, for a batch and on packed pages) -> ctx [B, H, Rv] fp16, the heads' contexts in latent space.

    q [B, H, 128] fp16.  q_positions None: q is rotated already (like `torch.ops.palu.decode_attn`'s); an int32 [B] tensor: q is
    not rotated, and these are its positions.  bfrag: `prepare_paged_b`.  seq_lens int32 [B] counts the cached rows of a sequence,
    the new token's own among them if it has been appended.  sm_scale defaults to 1 / sqrt(128).

    A sequence of length 0 gives zeros.  A length beyond the block table, or a page outside the pool within the length, gives NaN
    for that sequence; entries past the length are never read."""
    what = "paged_attn"
    _pool(pool, what)
    dev, G, P, Rk, Rv = pool.device, pool.num_groups, pool.page_size, pool.rank_k, pool.rank_v
    if not isinstance(q, torch.Tensor) or q.dtype != torch.float16 or q.device != dev:
        raise TypeError(f"{what}: q must be an fp16 tensor on the pool's device")
    if q.dim() != 3 or q.shape[2] != 128 or q.shape[1] % G:
        raise ValueError(f"{what}: q must be [B, H, 128] with H a multiple of the pool's {G} groups, got {tuple(q.shape)}")
    B, H, D = q.shape
    table = _int32(block_table, "block_table", 2, dev, what)
    lens = _int32(seq_lens, "seq_lens", 1, dev, what)
    qpos = None if q_positions is None else _int32(q_positions, "q_positions", 1, dev, what)
    M = table.shape[1]
    if table.shape[0] != B or lens.shape[0] != B or (qpos is not None and qpos.shape[0] != B):
        raise ValueError(f"{what}: block_table, seq_lens and q_positions must have one entry per query ({B})")
    lib = _lib.lib
    need = lib.palu_paged_b_bytes(H, G, Rk)
    if need == 0 or bfrag.dtype != torch.uint8 or bfrag.numel() != need or bfrag.device != dev or not bfrag.is_contiguous():
        raise ValueError(f"{what}: bfrag is not prepare_paged_b's layout of a B for H={H}, num_groups={G}, Rk={Rk} on {dev}")
    q = _rows16(q)
    ctx = torch.empty((B, H, Rv), dtype=torch.float16, device=dev)
    ws = torch.empty(lib.palu_paged_attn_workspace_bytes(B, H, G, M, P, Rk, Rv), dtype=torch.uint8, device=dev)
    inv = rope_inv_freq(dev, D, theta)
    _launch(dev, lib.palu_paged_attn_q4, "palu_paged_attn_q4", q.data_ptr(), q.stride(0), q.stride(1), bfrag.data_ptr(), *pool._ptrs,
            table.data_ptr(), table.stride(0), M, lens.data_ptr(), 0 if qpos is None else qpos.data_ptr(), inv.data_ptr(),
            ctx.data_ptr(), ws.data_ptr(), B, H, G, D, P, pool.num_pages, Rk, Rv, 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale))
    return ctx
