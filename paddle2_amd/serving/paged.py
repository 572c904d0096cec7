"""Paged-cache operators of the serving runtime: attention of new tokens over cache pages, and copies of pages.

Both run on hand-written kernels (csrc/kernels/chunk_attn.hip, csrc/kernels/kv_pages.hip) on the GPU; on CPU tensors the
same definitions run in PyTorch.  Inference only: nothing here records a gradient.
"""
from __future__ import annotations

import math
import operator

import torch

from ..framework.tensor import Tensor
from ..ops import _native as N

_HEAD_DIMS = (64, 128)
_CHUNK_WGS = 512        # workgroups that fit the chip at once
_CHUNK_MIN_KEYS = 256   # keys of a piece at least (128: the join costs more than the shorter pieces give)
_FEW_ROWS = 16          # rows (query heads of a kv head times new tokens) per sequence up to which they are few, on average;
                        # 8 times as many (128, a tile of many) in the longest there can be
_PAIR_TILES = 256       # tiles up to which two groups of waves share one (the CUs),
_PAIR_ROWS = 64         # if of 128 rows: where the sequences have that many, on average
_MAX_KEYS = 2**31 - 2**14   # positions are 32-bit, and a tile's loads reach past its last key


def _u(x):
    return x._t if isinstance(x, Tensor) else x


def _launch(dev, fn, *args):
    """fn(*args, stream) on ``dev``: its current stream, and it the current device meanwhile."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if dev.index == torch.cuda.current_device():
        fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            fn(*args, stream)


_INTS = (torch.int32, torch.int64, torch.int16, torch.uint8, torch.int8)


def _ints(t, name, rows, cols, dev):
    """An int tensor [rows] or (cols given) [rows, any] on ``dev`` as contiguous int32."""
    t = _u(t)
    if not torch.is_tensor(t) or t.dtype not in _INTS:
        raise TypeError(f"chunk_attention: {name} must be an integer tensor")
    if t.device != dev:
        raise ValueError(f"chunk_attention: {name} is on {t.device}, the queries on {dev}")
    shape = t.shape
    if len(shape) != (2 if cols else 1) or (rows is not None and shape[0] != rows):
        raise ValueError(f"chunk_attention: {name} has shape {tuple(shape)}, expected ({rows or 'B'}{', pages' if cols else ''})")
    if t.dtype is torch.int64:   # (what does not fit 32 bits stays as far out as it can)
        t = t.clamp(-2**31, 2**31 - 1)
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def chunk_attention(q, k_cache, v_cache, cu_seqlens_q, seq_lens, block_table=None, layout="paged", scale=None, out=None):
    """Attention of the new tokens of a ragged batch over a paged KV cache.

    q [T, Hq, D] holds the new tokens of all sequences back to back: sequence b owns rows cu_seqlens_q[b] ..
    cu_seqlens_q[b + 1] (int32 [B + 1], not decreasing).  seq_lens[b] (int32 [B]) counts the tokens of sequence b in the
    cache, these new ones included (write_kv comes first), so its new token i stands at position
    seq_lens[b] - n_b + i and sees the keys up to and including its own.  n_b may be 0, 1 (decoding) or any length, all in
    one call; the lengths are read on the device, so the call can be captured in a graph and replayed with others.

    Caches and ``block_table`` [B, max_blocks] as in :func:`decode_attention`: layout "paged" [num_blocks, block_size,
    Hk, D], "paddle_block" [num_blocks, Hk, block_size, D], "bhsd" [B, Hk, max_s, D] without a table.  A row that sees
    no key (position below 0) gives zeros; a page number outside the pool reads as zeros; lengths past the table are
    cut to it.  Rows past cu_seqlens_q[B] are left as they are in ``out`` and are undefined in a new output.

    With one token for every sequence it computes what decode_attention does (which takes other types too, by torch): in
    0.35 - 1.0 of its time where query heads share keys or there is one sequence, in 1.0 - 1.25 of it for 8 and more sequences
    of thousands of tokens with as many kv heads as query heads.

    bfloat16 and float16 with D 64 or 128 on the GPU, any Hq / Hk up to 128; K and V caches of the same strides, a page of
    less than 2^31 elements, rows of out and the caches 16-byte aligned (ValueError otherwise; queries that are not are
    copied).  Returns out [T, Hq, D]."""
    wrap = isinstance(q, Tensor)
    q, k_cache, v_cache, out = _u(q), _u(k_cache), _u(v_cache), _u(out)
    dev, dt, qs, ks = q.device, q.dtype, q.shape, k_cache.shape
    if len(qs) != 3 or len(ks) != 4 or ks != v_cache.shape:
        raise ValueError(f"chunk_attention: q {tuple(qs)}, caches {tuple(ks)}, {tuple(v_cache.shape)}")
    if k_cache.dtype is not dt or v_cache.dtype is not dt:
        raise TypeError(f"chunk_attention: q {dt}, caches {k_cache.dtype}, {v_cache.dtype}")
    if k_cache.device != dev or v_cache.device != dev:
        raise ValueError(f"chunk_attention: q on {dev}, caches on {k_cache.device}, {v_cache.device}")
    T, Hq, D = qs
    if layout == "paged":
        tok, head = 1, 2
    elif layout in ("paddle_block", "bhsd"):
        tok, head = 2, 1
    else:
        raise ValueError(f"chunk_attention: layout {layout!r}")
    bs, Hk = ks[tok], ks[head]
    if ks[3] != D or Hk == 0 or bs == 0 or Hq % Hk:
        raise ValueError(f"chunk_attention: q {tuple(qs)} does not fit the {layout} cache {tuple(ks)}")
    lens = _ints(seq_lens, "seq_lens", None, False, dev)
    B = lens.shape[0]
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", B + 1, False, dev)
    if layout == "bhsd":
        if ks[0] < B:
            raise ValueError(f"chunk_attention: {B} sequences, caches for {ks[0]}")
        table = torch.arange(B, dtype=torch.int32, device=dev)[:, None]
    elif block_table is None:
        raise ValueError(f"chunk_attention: layout {layout!r} needs a block_table")
    else:
        table = _ints(block_table, "block_table", B, True, dev)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"chunk_attention: scale {scale}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != qs or out.dtype is not dt or out.device != dev:
        raise ValueError(f"chunk_attention: out {tuple(out.shape)} {out.dtype} on {out.device}")
    if T and B:
        if dev.type == "cuda" and N.use_native(q):
            _chunk_native(q, k_cache, v_cache, cu, lens, table, tok, head, scale, out)
        else:
            with torch.no_grad():
                _chunk_reference(q, k_cache, v_cache, cu, lens, table, tok, scale, out)
    return Tensor._wrap(out) if wrap else out


def attend_chunk(q, k_cache, v_cache, cu_seqlens_q, seq_lens, block_table, layout="paged"):
    """chunk_attention of checked torch tensors, for the framework's own paths: by its PyTorch definition where the kernel
    does not take the type or the head dim, as decode_attention does."""
    Hk = k_cache.shape[2 if layout == "paged" else 1]
    if q.device.type != "cuda" or _kernel_takes(q, Hk):
        return chunk_attention(q, k_cache, v_cache, cu_seqlens_q, seq_lens, block_table, layout=layout)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    with torch.no_grad():
        _chunk_reference(q, k_cache, v_cache, cu_seqlens_q, seq_lens, block_table, 1 if layout == "paged" else 2,
                         1.0 / math.sqrt(q.shape[2]), out)
    return out


def _kernel_takes(q, Hk):
    return q.dtype in (torch.bfloat16, torch.float16) and q.shape[2] in _HEAD_DIMS and q.shape[1] <= 128 * Hk


def _chunk_native(q, kc, vc, cu, lens, table, tok, head, scale, out):
    T, Hq, D = q.shape
    B, max_blocks = table.shape
    ks, sk, so = kc.shape, kc.stride(), out.stride()
    bs, Hk = ks[tok], ks[head]
    G = Hq // Hk
    if not _kernel_takes(q, Hk):
        raise ValueError(f"chunk_attention: {q.dtype} with head dim {D} and {G} query heads per kv head (bfloat16 or float16, "
                         f"{_HEAD_DIMS}, at most 128)")
    if not max_blocks or not ks[0]:
        raise ValueError("chunk_attention: a cache or a block table without pages")
    if max_blocks * bs > _MAX_KEYS:
        raise ValueError(f"chunk_attention: a block table for {max_blocks * bs} tokens (at most {_MAX_KEYS})")
    if sk != vc.stride():
        raise ValueError("chunk_attention: the K and V caches have different strides")
    sq = q.stride()
    if sq[2] != 1 or (q.data_ptr() | sq[0] * 2 | sq[1] * 2) & 15:
        with torch.no_grad():
            q = q.clone(memory_format=torch.contiguous_format)
        sq = q.stride()
    pq, pk, pv, po = q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr()
    if sk[3] != 1 or so[2] != 1 or ((sk[0] | sk[1] | sk[2] | so[0] | so[1]) * 2 | pk | pv | po) & 15:
        raise ValueError("chunk_attention: the caches and out need contiguous, 16-byte aligned rows")
    rows, groups, splits = _chunk_plan(T, B, G, Hk, max_blocks * bs)
    # scratch of a split: the pieces' O, their (maximum, sum), and into how many a token's keys were split
    ws = torch.empty(splits * T * Hq * (D + 2) + T, dtype=torch.float32, device=q.device) if splits > 1 else None
    w0 = 0 if ws is None else ws.data_ptr()
    w1 = w0 + 4 * splits * T * Hq * D
    _launch(q.device, N.native().chunk_attn, int(q.dtype is torch.float16), pq, sq[0], sq[1], pk, pv, sk[0], sk[tok],
            sk[head], table.data_ptr(), max_blocks, ks[0], bs, cu.data_ptr(), lens.data_ptr(), po, so[0], so[1], B, T, Hq,
            Hk, D, rows, groups, splits, _CHUNK_MIN_KEYS, scale, w0, w1, w1 + 8 * splits * T * Hq)


def _chunk_plan(T, B, G, Hk, capacity):
    """Rows of a tile (16, or 128 and 16 for the sequences that have no more), groups of four waves that share one, and into
    how many pieces a tile's keys are split at most."""
    # Pieces of a tile's keys.  Two workgroups of four waves fit a CU: as many pieces as fit the chip at once.  Few rows
    # over many sequences: up to four rounds of smaller ones instead, since the lengths differ (64 x 8,000: 318 -> 295 us);
    # many rows are left whole, their pieces' O costs more than it evens out.
    longest = min(capacity // _CHUNK_MIN_KEYS, 64)
    # Few rows in every sequence, as far as the host can see: on average, and where all others bring one token the longest has
    # no more than a tile of many.  255 single tokens and a piece of 2,000, 32 heads, over 1,000 - 2,000: 1,990 us by tiles of
    # 16 and 1,190 with tiles of 128 beside them, 31 and one of 300: 429 and 325; the other way 32 x 2 tokens, 8 heads on 1,
    # over 2,000 - 4,000: 20 and 23, 32 x 4, 32 on 8: 90 and 93, 64 x 4: 184 and 170.
    if G <= 16 and T * G <= _FEW_ROWS * B and (T - B + 1) * G <= 8 * _FEW_ROWS:
        tiles = max(min(B, T), -(-T // (16 // G))) * Hk
        # No more tiles than CUs, but work for all: one workgroup of eight waves a CU, half as many pieces to join (8 x 4
        # tokens over 350 - 700, 32 heads: 18.9 us, with four waves 21.6; 1 over 16,000, 32 heads on 8: 24.8 and 31.6; the
        # other way 16 over 600 - 1,200, 32 on 8: 22.6 and 21.5).  With less work four waves: 1 over 1,400, 16 heads on 4,
        # takes 14.4 us, with eight 16.0.
        if tiles <= _PAIR_TILES < tiles * longest:
            return 16, 2, max(1, min(_CHUNK_WGS // 2 // tiles, longest))
        return 16, 1, max(1, min((_CHUNK_WGS if tiles < _CHUNK_WGS else 4 * _CHUNK_WGS) // tiles, longest))
    tiles = max(min(B, T), -(-T // (128 // G))) * Hk
    # No more tiles than CUs, parts of tiles at the sequences' ends counted: two groups of waves per tile, whose halves of
    # the keys are joined through LDS (700 tokens, 32 heads: 20 us, with one 29; 1,000 over 3,000, 32 heads on 8: 74 and 78;
    # 128 over 16,000, 16 on 4: 36 and 40; the other way 2 x 2,000 over 10,000, 8 on 1: 183 and 176).  With 512 tiles 2,048
    # tokens with nothing cached take 53.8 and 55.9, but 4 x 500 tokens 57 and 51, 4,096 tokens 169 and 152.  With 64 rows per
    # sequence no difference.
    most = N.native().chunk_attn_tiles(T, B, G, 128) * Hk
    groups = 2 if most <= _PAIR_TILES and T * G >= _PAIR_ROWS * B else 1
    return 128, groups, max(1, min(_CHUNK_WGS // (groups * tiles), longest))


def _chunk_reference(q, kc, vc, cu, lens, table, tok, scale, out):
    T, Hq, D = q.shape
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    if tok == 2:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    nb, bs, Hk = kc.shape[:3]
    cu, lens = cu.clamp(0, T).tolist(), lens.tolist()
    for b, L in enumerate(lens):
        q0, n = cu[b], cu[b + 1] - cu[b]
        if n <= 0:
            continue
        L = max(0, min(L, table.shape[1] * bs))
        j = torch.arange(L, device=q.device)
        page = table[b].long()[j // bs]
        ok = (page >= 0) & (page < nb)
        ks, vs = (torch.where(ok[:, None, None], c[page.clamp(0, nb - 1), j % bs], 0).to(acc) for c in (kc, vc))
        qs = q[q0:q0 + n].to(acc).reshape(n, Hk, Hq // Hk, D)
        hidden = j[None] > torch.arange(L - n, L, device=q.device)[:, None]
        s = torch.einsum("nhgd,lhd->hgnl", qs, ks) * scale
        s = s.masked_fill(hidden, float("-inf"))
        # rows that see no key: zeros.  Hidden values are left out, not multiplied by zero (they may be infinite)
        top = s.amax(-1, keepdim=True) if L else s.new_zeros(s.shape[:-1] + (1,))
        p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
        z = p.sum(-1, keepdim=True)
        bad = ~torch.isfinite(vs).all(-1).all(-1)
        o = torch.einsum("hgnl,lhd->nhgd", p, torch.where(bad[:, None, None], 0.0, vs))
        for i in bad.nonzero().flatten().tolist():
            first = max(0, i - (L - n))
            o[first:] += torch.einsum("hgn,hd->nhgd", p[:, :, first:, i], vs[i])
        z = z.permute(2, 0, 1, 3)
        out[q0:q0 + n] = torch.where(z == 0, 0.0, o / z).reshape(n, Hq, D).to(out.dtype)


def _check_pages(src, dst, blocks):
    """What the native library checks, for a host without it."""
    for t in (src, dst):
        if torch.is_tensor(t) or isinstance(t, str):
            raise TypeError(f"copy_kv_blocks: page numbers in a {type(t).__name__} (a sequence of integers)")
    src, dst = [operator.index(i) for i in src], [operator.index(i) for i in dst]
    if len(src) != len(dst):
        raise ValueError("src and dst differ in length")
    for i in src + dst:
        if not 0 <= i < blocks:
            raise ValueError(f"page {i} is not in the pool")
    if len(set(dst)) < len(dst):
        raise ValueError("a page is a destination twice")
    if set(src) & set(dst):
        raise ValueError("a page is both a source and a destination")


class KVBlockCopier:
    """Copies pages inside the K and V pools of all layers in one launch.

    ``k_caches`` / ``v_caches``: one tensor per layer, [num_blocks, ...], all of one shape, type, device and stride, each
    page contiguous.  The pools are checked once here and kept; ``copy`` may then be called as often as wanted, and checks
    them again when one's memory has been replaced."""

    def __init__(self, k_caches, v_caches):
        self._given = list(k_caches) + list(v_caches)
        self._wrapped = any(issubclass(c, Tensor) for c in set(map(type, self._given)))
        self.pools = [_u(t) for t in self._given] if self._wrapped else self._given
        self._check()

    def _check(self):
        pools = self.pools
        if not pools:
            raise ValueError("copy_kv_blocks: no caches")
        a = pools[0]
        if a.dim() < 2 or not a[:1].is_contiguous() or (a.shape[0] > 1 and a.stride(0) < a[0].numel()):
            raise ValueError("copy_kv_blocks: the pages of a cache must be contiguous")
        shape, dtype, device, stride = a.shape, a.dtype, a.device, a.stride()
        for t in pools:
            if t.shape != shape or t.dtype is not dtype or t.device != device or t.stride() != stride:
                raise ValueError("copy_kv_blocks: the caches differ in shape, type, device or stride")
        self._dev = a.device
        self._blocks = a.shape[0]
        self._bytes = (a.numel() // max(a.shape[0], 1)) * a.element_size()
        self._stride = a.stride(0) * a.element_size()
        self._native = self._dev.type == "cuda" and N.use_native(a)
        self._ptrs = [t.data_ptr() for t in pools]

    def copy(self, src, dst):
        """Page src[i] -> page dst[i] in every pool, on the current stream.  ``src`` / ``dst``: sequences of host integers
        (TypeError for others).  A page may be a source many times, a destination once, and never both; ValueError otherwise,
        with nothing copied."""
        if self._wrapped:
            self.pools = [_u(t) for t in self._given]
        if [t.data_ptr() for t in self.pools] != self._ptrs:
            self._check()
        self._checked_copy(src, dst)

    def _checked_copy(self, src, dst):
        if self._native:
            _launch(self._dev, N.native().kv_copy, self._ptrs, src, dst, self._blocks, self._bytes, self._stride)
            return
        (_check_pages if N.native() is None else N.native().kv_copy_check)(src, dst, self._blocks)
        if len(src):
            s, d = (torch.tensor(list(i), device=self._dev) for i in (src, dst))
            with torch.no_grad():
                for t in self.pools:
                    t[d] = t[s]


def copy_kv_blocks(k_caches, v_caches, src, dst):
    """``KVBlockCopier(k_caches, v_caches).copy(src, dst)``: page src[i] of every layer's K and V pool -> page dst[i].  A
    program that copies often keeps the copier (PagedKVCache.copy_blocks does)."""
    KVBlockCopier(k_caches, v_caches)._checked_copy(src, dst)
