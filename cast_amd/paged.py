"""A KV cache of pages: append with the rotation on the way, the attention of
one new token per request, and tree verification over it (HIP, gfx950).

  paged_append     rows of new K and V into their requests' pages, K (and Q)
                   rotated to their positions by cos / sin tables; the paged
                   form of cast_trees/serving.py:264-289
  paged_attention  one query token per request against the pages: the ordinary
                   decode step (cast_trees/decode.py:211-231 runs it inside the
                   model) beside the tree verification
  paged_tree_attention  cast_trees/tree_attn.py:116-139 with the prefix read out
                   of the pages, as store_tree_attention reads it out of a store

A layer's pool is ``[n_pages, Hkv, page_size, D]`` in bfloat16, float16 or
float32, with any strides of its first three dimensions that keep rows 16-byte
aligned (a ``[n_pages, page_size, Hkv, D]`` cache is passed as
``pool.transpose(1, 2)``).  Slot t of request b lies in page ``page_table[b, t
// page_size]`` at offset ``t % page_size``; ``page_table`` is int32 ``[B,
max_pages]``, entries behind a request's last page may be anything.  The
per-request store ``[B, Hkv, cap, D]`` of ``cast_amd.serving`` is such a pool of
one page per request: ``page_table = arange(B)[:, None]``.

Everything is stream-ordered on torch's current stream; nothing synchronises
unless ``check=True``, which reads the device status word once and raises
``ValueError``.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch

from . import _lib
from .tree_attn import _DTYPES, _as_i32, _host_side, _mask_words, _require_on, check_host_metadata


class _Pools:
    """A layer's pools as the launches need them, checked: sizes, addresses and
    strides (K's then V's), cast_dtype, element size and device index."""
    __slots__ = ("n_pages", "H_kv", "page_size", "D", "dtype", "code", "esz", "device", "index", "k", "v", "strides")

    def __init__(self, k_pages, v_pages, what):
        shape, dt = k_pages.shape, k_pages.dtype
        if len(shape) != 4 or v_pages.shape != shape:
            raise ValueError("k_pages and v_pages must both be [n_pages, H_kv, page_size, D]")
        self.n_pages, self.H_kv, self.page_size, self.D = shape
        self.index = k_pages.get_device()
        if self.index < 0:
            raise ValueError(f"{what} runs on the GPU: the pools must be device tensors")
        if dt not in _DTYPES or v_pages.dtype is not dt:
            raise ValueError("the pools must share one dtype: bfloat16, float16 or float32")
        self.dtype, self.code, self.esz, self.device = dt, _DTYPES[dt], dt.itemsize, k_pages.device
        ks, vs = k_pages.stride(), v_pages.stride()
        self.k, self.v = k_pages.data_ptr(), v_pages.data_ptr()
        self.strides = ks[:3] + vs[:3]
        low = self.k | self.v | (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) * self.esz
        if (ks[3] != 1 or vs[3] != 1 or low & 15) and self.n_pages:
            raise ValueError("the pools need a contiguous head dim and 16-byte aligned strides")
        if v_pages.get_device() != self.index:
            _require_on(self.device, v_pages=v_pages)


def _table(page_table, pools, batch=None):
    """page_table as int32 rows on the pools' device (no copy when it already is that)."""
    t = page_table
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == pools.index
            and t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] <= 1)):
        t = _as_i32(t, pools.device)
    if t.dim() != 2 or (batch is not None and t.shape[0] != batch):
        raise ValueError("page_table must be [B, max_pages]")
    return t


def _rows(name, x, heads, pools, total):
    """Check x as [total, heads, D] rows of the pools' dtype and device and
    return it, or a copy the kernels can address: head dim contiguous, 16-byte
    aligned base and strides."""
    if x.shape != (total, heads, pools.D):
        raise ValueError(f"{name} must be [{total}, {heads}, {pools.D}]")
    if x.dtype is not pools.dtype:
        raise ValueError(f"{name} must have the pools' dtype {pools.dtype}")
    if x.get_device() != pools.index:
        _require_on(pools.device, **{name: x})
    st = x.stride()
    if (st[2] == 1 and not (x.data_ptr() | (st[0] | st[1]) * pools.esz) & 15) or not x.numel():
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _output(name, x, heads, pools, total):
    """Check a caller's output like _rows; it is written where it lies."""
    if _rows(name, x, heads, pools, total) is not x:
        raise ValueError(f"{name} needs a contiguous head dim and 16-byte aligned strides")
    _no_overlap(name, x)
    return x


_INT32 = (1 << 31) - 1


def _workspace(workspace, need, like):
    """The caller's workspace where it holds `need` bytes, else a new one."""
    if workspace is not None:
        _require_on(like.device, workspace=workspace)
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace.numel() * workspace.element_size() >= need:
            return workspace
    return like.new_empty(need, dtype=torch.uint8)


def _no_overlap(name, t):
    """An output whose elements share memory (an expanded tensor) cannot be written."""
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} must not be an expanded tensor")


def paged_append(k, v, k_pages, v_pages, page_table, seq_len, cu_q=None, *, q=None, cos=None, sin=None,
                 positions=None, interleaved=False, q_out=None, k_out=None, new_len=None, check=False):
    """Write new tokens into the cache; returns ``(q_rotated, new_len)``.

    k / v: [total, H_kv, D] rows of the new tokens (any token and head
    strides); seq_len int32 [B]: tokens of each request already in the cache.
    Request b appends rows cu_q[b] .. cu_q[b + 1] - 1 (``cu_q=None``: one token
    each, row b) to slots seq_len[b], seq_len[b] + 1, ...  ``new_len`` int32 [B]
    (allocated unless given) is seq_len plus the rows appended.

    cos / sin: float32 [max_pos, rot_dim / 2]; with them the first rot_dim
    elements of every K head are rotated before they are stored: element pairs
    (i, i + rot_dim / 2), or (2i, 2i + 1) with ``interleaved``, by the angle of
    the token's slot or of ``positions`` int32 [total].  rot_dim: a multiple of
    16 (float32: of 8).  ``q`` [total, H_q, D] is rotated alike into ``q_out``
    (allocated unless given; may be q itself); without tables it is copied.
    ``k_out`` also receives the rotated K (may be k itself).

    A row with an invalid slot, page id or position is skipped whole, and its
    request's new_len stays seq_len; ``check=True`` raises.
    """
    if not check and k_pages.is_cuda:
        done = _lib.calls().paged_append(k, v, k_pages, v_pages, page_table, seq_len, cu_q, q, cos, sin, positions,
                                         interleaved, q_out, k_out, new_len, _lib.stream_of(k_pages))
        if type(done) is tuple:
            return done
        if done is not None:
            _lib.check(done, "cast_paged_append")
    # (a status to read, a copy to make, or something to refuse)
    lib = _lib.load()
    pools = _Pools(k_pages, v_pages, "paged_append")
    H_kv, D, dev, esz = pools.H_kv, pools.D, pools.device, pools.esz
    total = k.shape[0] if k.dim() else 0
    k, v = _rows("k", k, H_kv, pools, total), _rows("v", v, H_kv, pools, total)
    H_q = 0
    if q is not None:
        H_q = q.shape[1] if q.dim() == 3 else 0
        q = _rows("q", q, H_q, pools, total) if q_out is not q else _output("q", q, H_q, pools, total)
        assert H_q > 0 and H_q % H_kv == 0
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format) if q_out is None else \
            _output("q_out", q_out, H_q, pools, total)
        q_in, q_st, q_to, qo_st = q.data_ptr(), q.stride()[:2], q_out.data_ptr(), q_out.stride()[:2]
    elif q_out is not None:
        raise ValueError("q_out without q")
    else:
        q_in, q_to, q_st, qo_st = None, None, (0, 0), (0, 0)
    k_to, ko_st = (None, (0, 0)) if k_out is None else \
        (_output("k_out", k_out, H_kv, pools, total).data_ptr(), k_out.stride()[:2])
    rot_dim = max_pos = rope_ld = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
            raise ValueError("cos and sin must both be float32 [max_pos, rot_dim / 2]")
        max_pos, rot_dim = cos.shape[0], 2 * cos.shape[1]
        if not max_pos:
            raise ValueError("cos and sin hold no position")
        if not 0 < rot_dim <= D or rot_dim % (32 // esz):
            raise ValueError(f"rot_dim must be a multiple of {32 // esz} up to the head dim {D}, got {rot_dim}")
        if cos.get_device() != pools.index or sin.get_device() != pools.index:
            _require_on(dev, cos=cos, sin=sin)
        ld = cos.stride(0)
        if not (cos.is_contiguous() and sin.is_contiguous()) and (
                cos.stride() != sin.stride() or cos.stride(1) != 1 or ld % 4 or ld < rot_dim // 2):
            cos, sin = cos.contiguous(), sin.contiguous()
        if (cos.data_ptr() | sin.data_ptr()) & 15:
            cos, sin = cos.clone(), sin.clone()
        rope_ld = cos.stride(0) if max_pos > 1 else rot_dim // 2
        if positions is not None:
            positions = _as_i32(positions, dev)
            if positions.shape != (total,):
                raise ValueError(f"positions must be [{total}]")
    else:
        positions = None
    page_table = _table(page_table, pools)
    seq_len = _as_i32(seq_len, dev)
    B, max_pages = page_table.shape
    if seq_len.shape != (B,):
        raise ValueError(f"seq_len must be [{B}], one entry per page_table row")
    if cu_q is not None:
        cu_q = _as_i32(cu_q, dev)
        if cu_q.shape != (B + 1,):
            raise ValueError("cu_q needs B+1 entries")
    elif total != B:
        raise ValueError("without cu_q every request appends one row: k must have B rows")
    if new_len is None:
        new_len = torch.empty_like(seq_len)
    else:
        _require_on(dev, new_len=new_len)
        if new_len.dtype is not torch.int32 or new_len.shape != (B,) or not new_len.is_contiguous():
            raise ValueError(f"new_len must be a contiguous int32 [{B}]")
    if not total:
        new_len.copy_(seq_len)      # nothing to append
        return q_out, new_len
    status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    one = lambda address: ctypes.byref(ctypes.c_void_p(address))
    with _lib.on_device(dev):
        st = lib.cast_paged_append(
            one(k.data_ptr()), one(v.data_ptr()), one(pools.k), one(pools.v), 1, page_table.data_ptr(),
            page_table.stride(0), max_pages, pools.n_pages, pools.page_size, seq_len.data_ptr(), new_len.data_ptr(), B,
            total, _lib.ptr(cu_q), None, 0, None, q_in, q_to, k_to, _lib.ptr(cos), _lib.ptr(sin), rope_ld, max_pos,
            rot_dim, 1 if interleaved else 0, _lib.ptr(positions), H_q, H_kv, D, *k.stride()[:2], *v.stride()[:2],
            *pools.strides, *q_st, *qo_st, *ko_st, pools.code, _lib.ptr(status), _lib.stream_of(k_pages))
    _lib.check(st, "cast_paged_append")
    if check:
        _lib.raise_device_flags(status.item(), "paged_append")
    return q_out, new_len


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device_index, *sizes):
    """cast_paged_attn_workspace_size of one call's sizes, asked once per size
    with the device current (plain ints: a function of them alone)."""
    with _lib.on_device(torch.device("cuda", device_index)):
        return _lib.load().cast_paged_attn_workspace_size(*sizes)


def paged_attention(q, k_pages, v_pages, page_table, seq_len, sm_scale=None, *, softcap=0.0, window=0,
                    return_lse=False, kv_split=0, check=False, out=None, workspace=None):
    """q: [B, H_q, D], one new token per request -> [B, H_q, D].

    seq_len int32 [B]: slots request b's query sees, its own token's included
    (0 gives zeros and lse = -inf).  Scores are ``sm_scale * q.k`` (default
    1 / sqrt(D)), capped to ``softcap * tanh(score / softcap)`` when softcap is
    positive; with ``window > 0`` only the last ``window`` slots are seen.
    ``return_lse`` also returns their natural-log log-sum-exp [B, H_q] (fp32).
    ``kv_split``: keys per split of a request (0: chosen on the device from the
    lengths, none where table rows or the window are short; negative: none).  ``workspace``: uint8 device tensor of at
    least ``paged_workspace_bytes(...)``; one is allocated when missing or too
    small.  Calls that share a workspace must not overlap.

    Requests with a length outside the table or a visible page id outside the
    pool return zeros with lse = -inf; ``check=True`` raises.
    """
    # (sizes past 31 bits mean what the largest of them does)
    kv_split, window = max(-1, min(operator.index(kv_split), _INT32)), min(operator.index(window), _INT32)
    if not check and k_pages.is_cuda:
        done = _lib.calls().paged_attention(q, k_pages, v_pages, page_table, seq_len, sm_scale, softcap, window, kv_split,
                                            return_lse, out, workspace, _lib.stream_of(k_pages))
        if type(done) is int:
            _lib.check(done, "cast_paged_attn_fwd")
        if done is not None:
            return done
    # (a status to read, a copy to make, or something to refuse)
    lib = _lib.load()
    pools = _Pools(k_pages, v_pages, "paged_attention")
    H_kv, D, dev = pools.H_kv, pools.D, pools.device
    if q.dim() != 3:
        raise ValueError(f"q must be [B, H_q, {D}]")
    B, H_q, _ = q.shape
    assert H_q % H_kv == 0
    q = _rows("q", q, H_q, pools, B)
    if window < 0 or not 0 <= softcap < math.inf:
        raise ValueError("window and softcap must be 0 (none) or positive")
    page_table = _table(page_table, pools, B)
    seq_len = _as_i32(seq_len, dev)
    if seq_len.shape != (B,):
        raise ValueError(f"seq_len must be [{B}]")
    out = q.new_empty((B, H_q, D)) if out is None else _output("out", out, H_q, pools, B)
    lse = q.new_empty((B, H_q), dtype=torch.float32) if return_lse else None
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    max_pages = page_table.shape[1]
    ws_bytes = _workspace_bytes(pools.index, B, max_pages, pools.page_size, H_q, H_kv, D, window, pools.code, kv_split)
    if ws_bytes or workspace is not None:
        workspace = _workspace(workspace, ws_bytes, q)
    status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    with _lib.on_device(dev):
        st = lib.cast_paged_attn_fwd(
            q.data_ptr(), pools.k, pools.v, out.data_ptr(), _lib.ptr(lse), page_table.data_ptr(), page_table.stride(0),
            max_pages, pools.n_pages, pools.page_size, seq_len.data_ptr(), B, H_q, H_kv, D, *q.stride()[:2],
            *pools.strides, *out.stride()[:2], pools.code, float(sm_scale), float(softcap), window, kv_split,
            workspace.data_ptr() if ws_bytes else None, ws_bytes, _lib.ptr(status), _lib.stream_of(q))
    _lib.check(st, "cast_paged_attn_fwd")
    if check:
        _lib.raise_device_flags(status.item(), "paged_attention")
    return (out, lse) if return_lse else out


def paged_workspace_bytes(batch, max_pages, page_size, H_q, H_kv, D, dtype=torch.bfloat16, window=0, kv_split=0,
                          device=None):
    """Bytes of split workspace one ``paged_attention`` call of these sizes needs."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return _workspace_bytes(dev.index or 0, batch, max_pages, page_size, H_q, H_kv, D, window, _DTYPES[dtype], kv_split)


@functools.lru_cache(maxsize=256)
def _tree_workspace_bytes(device_index, *sizes):
    """cast_tree_attn_paged_workspace_size of one call's sizes, with the device current."""
    with _lib.on_device(torch.device("cuda", device_index)):
        return _lib.load().cast_tree_attn_paged_workspace_size(*sizes)


def paged_tree_workspace_bytes(q, k_pages, page_table, total_kv, kv_split=0):
    """Bytes of workspace one ``paged_tree_attention`` call of these tensors needs."""
    total_q, H_q, D = q.shape
    return _tree_workspace_bytes(k_pages.device.index, int(page_table.shape[0]), total_q, int(total_kv), H_q,
                                 int(k_pages.shape[1]), D, _DTYPES[k_pages.dtype], kv_split)


def paged_tree_attention(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len, pack_len, ancestor_mask,
                         sm_scale=None, *, total_kv=None, return_lse=False, kv_split=0, check=False, out=None,
                         workspace=None):
    """Tree-verification attention whose prefix lies in pages.

    The attention of ``cast_amd.tree_attn.store_tree_attention``, with the same
    bits over the same tokens: request b's keys are slots [0, prefix_len[b]) of
    its pages followed by its pack.

      q              [total_q, H_q, D]  (any token/head strides)
      k_pages/v_pages  pools [n_pages, H_kv, page_size, D], page_size a multiple
                     of 64 (any size where page_table has one column)
      k_pack/v_pack  [H_kv, total_q, D] the pass's own K/V
      total_kv       host bound on sum(prefix_len + pack_len) that sizes launch
                     and workspace (default B * max_pages * page_size + total_q)

    Returns ``out`` [total_q, H_q, D] (and ``lse`` with ``return_lse``).  A
    request whose prefix names a page outside the pool is rejected like one with
    inconsistent lengths: zeros with lse = -inf, and ``check=True`` raises.
    """
    kv_split = max(-_INT32, min(operator.index(kv_split), _INT32))
    if not check and k_pages.is_cuda:
        done = _lib.calls().paged_tree_attention(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len, pack_len,
                                                 ancestor_mask, sm_scale, total_kv, return_lse, kv_split, out, workspace,
                                                 _lib.stream_of(k_pages))
        if type(done) is int:
            _lib.check(done, "cast_tree_attn_paged_fwd")
        if done is not None:
            return done
    # (a status to read, a copy to make, or something to refuse)
    lib = _lib.load()
    pools = _Pools(k_pages, v_pages, "paged_tree_attention")
    H_kv, D, dev = pools.H_kv, pools.D, pools.device
    if pools.n_pages == 0:
        raise ValueError("the pools must hold at least one page")
    if q.dim() != 3:
        raise ValueError(f"q must be [total_q, H_q, {D}]")
    total_q, H_q, _ = q.shape
    assert H_q % H_kv == 0
    q = _rows("q", q, H_q, pools, total_q)
    if k_pack.dim() != 3 or v_pack.dim() != 3:
        raise ValueError(f"k_pack/v_pack must be [{H_kv}, {total_q}, {D}]")
    kn = _rows("k_pack (token-major)", k_pack.transpose(0, 1), H_kv, pools, total_q)
    vn = _rows("v_pack (token-major)", v_pack.transpose(0, 1), H_kv, pools, total_q)
    page_table = _table(page_table, pools)
    B, max_pages = page_table.shape
    if pools.page_size % 64 and max_pages > 1:
        raise ValueError("paged_tree_attention needs a page size that is a multiple of 64")
    total_kv = B * max_pages * pools.page_size + total_q if total_kv is None else operator.index(total_kv)
    if not 0 <= total_kv < 1 << 31:
        raise ValueError("total_kv must be a bound on the summed lengths below 2^31")
    mask, words = _mask_words(ancestor_mask, total_q, dev)
    if _host_side(cu_q, prefix_len, pack_len):
        check_host_metadata(cu_q, prefix_len, pack_len, total_q, total_kv, words, cap=max_pages * pools.page_size)
    cu_q, prefix_len, pack_len = _as_i32(cu_q, dev), _as_i32(prefix_len, dev), _as_i32(pack_len, dev)
    if cu_q.shape != (B + 1,) or prefix_len.shape != (B,) or pack_len.shape != (B,):
        raise ValueError("cu_q needs B+1 entries and prefix_len / pack_len B entries (B rows of page_table)")
    out = q.new_empty((total_q, H_q, D)) if out is None else _output("out", out, H_q, pools, total_q)
    lse = q.new_empty((total_q, H_q), dtype=torch.float32) if return_lse else None
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    ws_bytes = _tree_workspace_bytes(pools.index, B, total_q, total_kv, H_q, H_kv, D, pools.code, kv_split)
    workspace = _workspace(workspace, ws_bytes, q)
    status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    with _lib.on_device(dev):
        st = lib.cast_tree_attn_paged_fwd(
            q.data_ptr(), pools.k, pools.v, page_table.data_ptr(), page_table.stride(0), max_pages, pools.n_pages,
            pools.page_size, kn.data_ptr(), vn.data_ptr(), out.data_ptr(), _lib.ptr(lse), cu_q.data_ptr(),
            prefix_len.data_ptr(), pack_len.data_ptr(), mask.data_ptr(), words, B, total_q, total_kv, H_q, H_kv, D,
            *q.stride()[:2], *pools.strides, *kn.stride()[:2], *vn.stride()[:2], *out.stride()[:2], pools.code,
            float(sm_scale), kv_split, workspace.data_ptr(), ws_bytes, _lib.ptr(status), _lib.stream_of(q))
    _lib.check(st, "cast_tree_attn_paged_fwd")
    if check:
        _lib.raise_device_flags(status.item(), "paged_tree_attention")
    return (out, lse) if return_lse else out
