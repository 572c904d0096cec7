"""Chunk attention over a paged cache, page copies and token sampling against plain 64-bit forms, their refusals, and a
run of them together through the cache and the generator.  CPU tensors take the PyTorch definitions; the gpu-marked
tests take the HIP kernels."""
import math

import pytest
import torch

import paddle2_amd as paddle
from paddle2_amd import serving
from paddle2_amd.ops import _native as N


# ============================================================================ chunk attention
def _batch(dev, dtype, new, held, Hq, Hk, D, bs, layout="paged", seed=0, extra_rows=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    lens = [n + h for n, h in zip(new, held)]
    need = [max(0, -(-L // bs)) for L in lens]
    nb = sum(need) + spare
    perm = torch.randperm(nb, generator=g).tolist()
    table = torch.zeros(len(new), max(need + [1]), dtype=torch.int32)
    for b, k in enumerate(need):
        table[b, :k] = torch.tensor([perm.pop() for _ in range(k)], dtype=torch.int32)
    shape = (nb, bs, Hk, D) if layout == "paged" else (nb, Hk, bs, D)
    kc = torch.randn(shape, generator=g).to(dtype)
    vc = torch.randn(shape, generator=g).to(dtype)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1] + extra_rows, Hq, D, generator=g) * 1.5).to(dtype)
    return [t.to(dev) for t in (q, kc, vc, torch.tensor(cu, dtype=torch.int32),
                                torch.tensor(lens, dtype=torch.int32), table)]


def _attn64(q, kc, vc, cu, lens, table, layout="paged", scale=None):
    """(o, sum p |v| / sum p, largest sum |q k| scale) per row in 64 bits; rows without keys are zeros."""
    q, kc, vc = (t.double().cpu() for t in (q, kc, vc))
    if layout == "paddle_block":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    nb, bs, Hk, D = kc.shape
    cu, lens, table = cu.tolist(), lens.tolist(), table.cpu()
    G = q.shape[1] // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    o, a, big = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2])
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        L = min(L, table.shape[1] * bs)
        pages = table[b].long()
        ok = (pages >= 0) & (pages < nb)
        K = (kc[pages.clamp(0, nb - 1)] * ok[:, None, None, None]).reshape(-1, Hk, D)[:L]
        V = torch.where(ok[:, None, None, None], vc[pages.clamp(0, nb - 1)], 0.0).reshape(-1, Hk, D)[:L]
        for i in range(n):
            p = L - n + i + 1
            if p <= 0:
                continue
            for h in range(q.shape[1]):
                z = K[:p, h // G] @ q[cu[b] + i, h] * scale
                w = torch.softmax(z, 0)
                o[cu[b] + i, h] = w @ V[:p, h // G]
                a[cu[b] + i, h] = w @ V[:p, h // G].abs()
                big[cu[b] + i, h] = (K[:p, h // G].abs() @ q[cu[b] + i, h].abs()).max() * scale
    return o, a, big


def _tolerance(dtype, D, o, a, big):
    """Half a step for the output and for every 16-bit weight; scores summed in 32 bits over D products, scaled and
    exponentiated with one rounding each, move a weight by (D + 8) half steps of the largest sum of |q k|."""
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    move = torch.expm1((D + 8) * 2.0 ** -24 * (big.double() + 1))[..., None]
    return 1.01 * half * (o.abs() + a) + 2.02 * move * a + 2.0 ** -22 * a + 1e-7


def _check_attn(dev, dtype, new, held, Hq, Hk, D, bs, layout="paged", **kw):
    case = _batch(dev, dtype, new, held, Hq, Hk, D, bs, layout, **kw)
    out = serving.chunk_attention(*case, layout=layout)
    o, a, big = _attn64(*case, layout=layout)
    T = int(case[3][-1])
    assert ((out[:T].double().cpu() - o[:T]).abs() <= _tolerance(dtype, D, o, a, big)[:T]).all()
    return case, out


ATTN = [  # new, held, Hq, Hk, D, block
    ([1], [0], 4, 4, 64, 16),
    ([1, 1, 1], [0, 62, 63], 8, 2, 128, 16),
    ([5], [0], 4, 1, 128, 16),
    ([64], [0], 2, 2, 128, 64),
    ([65, 1, 128], [0, 200, 63], 4, 2, 64, 32),
    ([3, 0, 17, 1], [500, 33, 0, 0], 8, 1, 128, 16),
    ([7], [1000], 12, 4, 64, 24),          # three heads per group, pages of 24 tokens
    ([33, 2], [95, 1], 14, 2, 128, 5),     # seven heads per group, pages of 5 tokens
    ([130], [129], 5, 1, 64, 128),
    ([16, 16], [700, 1], 16, 1, 128, 64),
    ([2], [3], 128, 1, 64, 16),            # one token per row tile
    ([2], [70], 70, 1, 64, 16),
]


@pytest.mark.parametrize("layout", ["paged", "paddle_block"])
@pytest.mark.parametrize("case", ATTN[:7], ids=str)
def test_chunk_attention_cpu(case, layout):
    _check_attn("cpu", torch.float32, *case, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["paged", "paddle_block"])
@pytest.mark.parametrize("case", ATTN, ids=str)
def test_chunk_attention_gpu(case, layout, dtype):
    _check_attn("cuda", dtype, *case, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(4, 4), (8, 2), (16, 1)])
@pytest.mark.parametrize("new,held", [([1, 2, 300], [4000, 2001, 1700]), ([600], [1500]), ([9, 16, 17, 33], [5, 0, 3001, 777])])
def test_chunk_attention_long_gpu(new, held, Hq, Hk, D):
    _check_attn("cuda", torch.bfloat16, new, held, Hq, Hk, D, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,pairs", [(0, 0), (0, 10 ** 6), (10 ** 6, 0), (10 ** 6, 1000)])
@pytest.mark.parametrize("splits", [1, 10 ** 6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunk_attention_every_kernel_gpu(rows, pairs, splits, dtype, monkeypatch):
    """The kernels for few rows and for many, one group of waves or two per tile, with the keys in one piece and in as many
    as possible, on the same batches."""
    from paddle2_amd.serving import paged

    plan = paged._chunk_plan
    if pairs == 1000:       # two groups whatever the work
        monkeypatch.setattr(paged, "_chunk_plan", lambda *a: (16, 2, 1 if splits == 1 else plan(*a)[2]))
    monkeypatch.setattr(paged, "_FEW_ROWS", rows)
    monkeypatch.setattr(paged, "_PAIR_TILES", pairs)
    monkeypatch.setattr(paged, "_PAIR_ROWS", 0)
    monkeypatch.setattr(paged, "_CHUNK_WGS", splits)
    for D in (64, 128):
        _check_attn("cuda", dtype, [1, 0, 40, 3], [1000, 50, 700, 0], 8, 2, D, 16)
        _check_attn("cuda", dtype, [2, 17], [129, 400], 4, 4, D, 32, seed=1)
        _check_attn("cuda", dtype, [9, 1], [127, 255], 6, 2, D, 12, seed=2)
        _check_attn("cuda", dtype, [5, 4], [300, 31], 16, 1, D, 7, seed=3)
        q, kc, vc, cu, lens, table = _batch("cuda", dtype, [10, 4], [0, 600], 4, 1, D, 16, seed=4)
        lens[0] = 4
        assert (serving.chunk_attention(q, kc, vc, cu, lens, table)[:6] == 0).all()
        for bad in (float("nan"), float("inf")):      # behind token 2 of sequence 1: its last token alone sees it
            good = serving.chunk_attention(q, kc, vc, cu, lens, table)
            vc[table[1, 603 // 16].long(), 603 % 16] = bad
            out = serving.chunk_attention(q, kc, vc, cu, lens, table)
            torch.testing.assert_close(out[:13], good[:13], rtol=2 ** -7, atol=1e-3)
            assert not torch.isfinite(out[13]).any()
            vc[table[1, 603 // 16].long(), 603 % 16] = 1.0


@pytest.mark.gpu
def test_chunk_attention_many_sequences_gpu():
    """More sequences than a wave has lanes, lengths of zero among them."""
    new = [(i * 7) % 5 for i in range(150)]
    held = [(i * 13) % 90 for i in range(150)]
    _check_attn("cuda", torch.bfloat16, new, held, 4, 2, 64, 16)
    for i in range(3, 150, 11):      # pieces of prompts among them: both kinds of tiles in one launch
        new[i] = 40 + i % 60
    for D in (64, 128):
        _check_attn("cuda", torch.float16, new, held, 4, 2, D, 16, seed=D)
    _check_attn("cuda", torch.bfloat16, new, held, 34, 1, 64, 16)      # more heads than a tile of few rows has rows


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_chunk_attention_rows_without_keys_and_bad_pages(dev):
    """More new tokens than the cache holds: the first rows see nothing and give zeros.  Page numbers outside the pool
    read as zeros.  Lengths past the table are cut to it."""
    dt = torch.float32 if dev == "cpu" else torch.bfloat16
    q, kc, vc, cu, lens, table = _batch(dev, dt, [10, 40, 3], [0, 60, 20], 4, 2, 64, 16)
    lens[0] = 4
    lens[2] = 10 ** 9
    table[1, 2], table[1, 4] = -1, kc.shape[0]
    out = serving.chunk_attention(q, kc, vc, cu, lens, table)
    assert (out[:6] == 0).all() and (out[6] != 0).any()
    o, a, big = _attn64(q, kc, vc, cu, lens, table)
    assert ((out.double().cpu() - o).abs() <= _tolerance(dt, 64, o, a, big)).all()
    lens[1] = 0
    assert (serving.chunk_attention(q, kc, vc, cu, lens, table)[10:50] == 0).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_chunk_attention_hidden_values_do_not_matter(dev, bad):
    """NaN and infinities in the unused rest of a sequence's pages, in other pages, and in new tokens behind a row."""
    dt = torch.float32 if dev == "cpu" else torch.float16
    new, held = [70, 5, 1], [10, 300, 33]
    q, kc, vc, cu, lens, table = _batch(dev, dt, new, held, 4, 2, 64, 16)
    good = serving.chunk_attention(q, kc, vc, cu, lens, table)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, L in enumerate(lens.tolist()):
        j = torch.arange(L)
        used[table[b].cpu().long()[j // 16], j % 16] = True
    kc[~used.to(dev)] = bad
    vc[~used.to(dev)] = bad
    out = serving.chunk_attention(q, kc, vc, cu, lens, table)
    assert torch.equal(out, good)
    # token 50 of sequence 0 (position 60) and the last of sequence 1: rows before them stay as they were
    for b, p in ((0, 60), (1, 304)):
        kc[table[b, p // 16].long(), p % 16] = bad
        vc[table[b, p // 16].long(), p % 16, :, 3] = bad
    out = serving.chunk_attention(q, kc, vc, cu, lens, table)
    keep = [i for i in range(76) if not (50 <= i < 70 or i == 74)]
    torch.testing.assert_close(out[keep], good[keep], rtol=2 ** -10, atol=1e-3 if dev == "cuda" else 1e-6)
    assert not torch.isfinite(out[50:70, :, 3]).any()


@pytest.mark.gpu
def test_chunk_attention_infinite_values_that_are_seen_gpu():
    """A visible infinity makes its column infinite, opposite ones make it NaN, other columns stay."""
    q, kc, vc, cu, lens, table = _batch("cuda", torch.bfloat16, [40], [0], 2, 1, 64, 16)
    good = serving.chunk_attention(q, kc, vc, cu, lens, table)
    inf = float("inf")
    vc[table[0, 0].long(), 5, 0, 7] = inf
    vc[table[0, 1].long(), 4, 0, 7] = -inf     # position 20
    vc[table[0, 0].long(), 9, 0, 8] = -inf
    out = serving.chunk_attention(q, kc, vc, cu, lens, table).float()
    assert (out[5:20, :, 7] == inf).all() and out[20:, :, 7].isnan().all() and (out[9:, :, 8] == -inf).all()
    rest = [d for d in range(64) if d not in (7, 8)]
    torch.testing.assert_close(out[:, :, rest], good[:, :, rest].float(), rtol=2 ** -7, atol=1e-3)
    torch.testing.assert_close(out[:5], good[:5].float(), rtol=2 ** -7, atol=1e-3)


@pytest.mark.gpu
def test_chunk_attention_strides_and_out_gpu():
    """q and out as views of wider rows, caches as layers of one allocation; rows past the last sequence stay."""
    q, kc, vc, cu, lens, table = _batch("cuda", torch.bfloat16, [20, 3], [50, 0], 8, 2, 64, 16, extra_rows=4)
    ref = serving.chunk_attention(q, kc, vc, cu, lens, table)
    wide = torch.zeros(q.shape[0], 12, 64, dtype=q.dtype, device="cuda")
    wide[:, 2:10] = q
    pool = torch.zeros(2, 3, *kc.shape, dtype=q.dtype, device="cuda")
    pool[0, 1], pool[1, 1] = kc, vc
    out = torch.full((q.shape[0], 16, 64), 7.0, dtype=q.dtype, device="cuda")
    got = serving.chunk_attention(wide[:, 2:10], pool[0, 1], pool[1, 1], cu.long(), lens.long(), table.long(),
                                  out=out[:, 4:12])
    assert got.data_ptr() == out[:, 4:12].data_ptr()
    assert torch.equal(out[:23, 4:12], ref[:23]) and (out[23:] == 7).all() and (out[:, :4] == 7).all()
    shifted = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)   # 2-byte aligned queries
    shifted.copy_(q)
    assert torch.equal(serving.chunk_attention(shifted, kc, vc, cu, lens, table)[:23], ref[:23])
    t = serving.chunk_attention(paddle.Tensor._wrap(q), paddle.Tensor._wrap(kc), paddle.Tensor._wrap(vc),
                                paddle.Tensor._wrap(cu), paddle.Tensor._wrap(lens), paddle.Tensor._wrap(table))
    assert isinstance(t, paddle.Tensor) and torch.equal(t._t[:23], ref[:23])


@pytest.mark.gpu
def test_chunk_attention_contiguous_caches_gpu():
    """layout "bhsd": every sequence's keys in one row of the cache."""
    g = torch.Generator().manual_seed(3)
    q = torch.randn(9, 4, 64, generator=g).cuda().bfloat16()
    kc, vc = (torch.randn(3, 2, 77, 64, generator=g).cuda().bfloat16() for _ in range(2))
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    lens = torch.tensor([77, 30], dtype=torch.int32, device="cuda")
    out = serving.chunk_attention(q, kc, vc, cu, lens, layout="bhsd")
    table = torch.arange(2, dtype=torch.int32, device="cuda")[:, None]
    o, a, big = _attn64(q, kc, vc, cu, lens, table, layout="paddle_block")
    assert ((out.double().cpu() - o).abs() <= _tolerance(torch.bfloat16, 64, o, a, big)).all()


@pytest.mark.gpu
def test_chunk_attention_far_pages_gpu():
    """Pages whose elements lie past 2^31."""
    bs, Hk, D = 64, 8, 128
    nb = 2 ** 31 // (bs * Hk * D) + 40
    kc = torch.zeros(nb, bs, Hk, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    q, k1, v1, cu, lens, table = _batch("cuda", torch.bfloat16, [5, 1], [900, 1200], 8, 8, 128, 64)
    ref = serving.chunk_attention(q, k1, v1, cu, lens, table)
    at = nb - k1.shape[0]
    kc[at:], vc[at:] = k1, v1
    assert torch.equal(serving.chunk_attention(q, kc, vc, cu, lens, table + at), ref)


@pytest.mark.gpu
def test_chunk_attention_captured_gpu():
    """A captured call follows new lengths, tables and values; two graphs and the eager path do not share scratch."""
    cases = [_batch("cuda", torch.bfloat16, [4, 1, 7], h, 8, 2, 128, 16, seed=i, spare=200 - i)
             for i, h in enumerate(([300, 20, 0], [800, 3, 64], [100, 700, 33]))]
    nb = max(c[1].shape[0] for c in cases)
    mb = max(c[5].shape[1] for c in cases)

    def fit(c):
        q, kc, vc, cu, lens, table = c
        pad = lambda t: torch.cat([t, torch.zeros(nb - t.shape[0], *t.shape[1:], dtype=t.dtype, device="cuda")])  # noqa: E731
        return [q, pad(kc), pad(vc), cu, lens, torch.nn.functional.pad(table, (0, mb - table.shape[1]))]

    cases = [fit(c) for c in cases]
    want = [serving.chunk_attention(*c) for c in cases]
    graphs = []
    for i in range(2):
        static = [t.clone() for t in cases[i]]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            serving.chunk_attention(*static)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = serving.chunk_attention(*static)
        graphs.append((g, static, out))
    for turn in range(4):
        for j, (g, static, out) in enumerate(graphs):
            i = (turn + j) % 3
            for a, b in zip(static, cases[i]):
                a.copy_(b)
            g.replay()
            eager = serving.chunk_attention(*cases[i])
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]) and torch.equal(eager, want[i])


@pytest.mark.gpu
def test_chunk_attention_other_stream_gpu():
    case = _batch("cuda", torch.bfloat16, [50, 2], [100, 3000], 8, 2, 128, 64)
    want = serving.chunk_attention(*case)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = serving.chunk_attention(*case)
    s.synchronize()
    assert torch.equal(got, want)


def _refused(dev, dt):
    q, kc, vc, cu, lens, table = _batch(dev, dt, [3, 2], [5, 1], 4, 2, 64, 16)
    call = serving.chunk_attention
    bad = [
        (ValueError, lambda: call(q[0], kc, vc, cu, lens, table)),
        (ValueError, lambda: call(q, kc, vc[:-1], cu, lens, table)),
        (TypeError, lambda: call(q, kc.double(), vc.double(), cu, lens, table)),
        (ValueError, lambda: call(q[:, :3], kc, vc, cu, lens, table)),
        (ValueError, lambda: call(q[..., :32], kc, vc, cu, lens, table)),
        (ValueError, lambda: call(q, kc, vc, cu[:-1], lens, table)),
        (ValueError, lambda: call(q, kc, vc, cu, lens, table[:1])),
        (TypeError, lambda: call(q, kc, vc, cu.float(), lens, table)),
        (ValueError, lambda: call(q, kc, vc, cu, lens)),
        (ValueError, lambda: call(q, kc, vc, cu, lens, table, layout="rows")),
        (ValueError, lambda: call(q, kc, vc, cu, lens, table, scale=0.0)),
        (ValueError, lambda: call(q, kc, vc, cu, lens, table, out=q[:2].clone())),
        (ValueError, lambda: call(q, kc, vc, cu, lens, layout="bhsd", out=q.float())),
    ]
    for err, f in bad:
        with pytest.raises(err):
            f()


def test_chunk_attention_refusals_cpu():
    _refused("cpu", torch.float32)
    m = N.native()
    with pytest.raises(ValueError):
        m.chunk_attn_tiles(4, 1, 129, 128)
    with pytest.raises(ValueError):
        m.chunk_attn_tiles(4, 1, 17, 16)
    # enough tiles for every split of T rows over B sequences
    for T in (1, 5, 2048):
        for B in (1, 3, 64):
            for rows, Gs in ((128, (1, 3, 128)), (16, (1, 3, 16))):
                for G in Gs:
                    per, some = rows // G, min(B, T)
                    most = some + (T - some) // per        # `some` sequences of one row, the rest in full tiles
                    assert most <= m.chunk_attn_tiles(T, B, G, rows) <= most + some


@pytest.mark.gpu
def test_chunk_attention_refusals_gpu():
    _refused("cuda", torch.bfloat16)
    q, kc, vc, cu, lens, table = _batch("cuda", torch.bfloat16, [3], [5], 4, 2, 64, 16)
    for f in (lambda: serving.chunk_attention(q.float(), kc.float(), vc.float(), cu, lens, table),
              lambda: serving.chunk_attention(q[..., :32].contiguous(), kc[..., :32].contiguous(),
                                              vc[..., :32].contiguous(), cu, lens, table),
              lambda: serving.chunk_attention(q, kc, vc, cu.cpu(), lens, table),
              lambda: serving.chunk_attention(q, kc, vc.cpu(), cu, lens, table),
              lambda: serving.chunk_attention(q, kc[:1].repeat(1, 4096, 1, 1), vc[:1].repeat(1, 4096, 1, 1), cu, lens,
                                              torch.zeros(1, 2 ** 15, dtype=torch.int32, device="cuda")),
              lambda: serving.chunk_attention(q, kc, vc.transpose(1, 2).contiguous().transpose(1, 2), cu, lens, table)):
        with pytest.raises(ValueError):
            f()
    assert serving.chunk_attention(q[:0], kc, vc, cu * 0, lens, table).shape == (0, 4, 64)


# ============================================================================ page copies
PAGES = [  # pools, blocks, page shape, type, pairs, sources
    (1, 4, (16, 2, 64), torch.bfloat16, 1, 1),
    (2, 40, (16, 1, 64), torch.float16, 17, 3),
    (3, 900, (1, 1, 8), torch.bfloat16, 400, 400),     # more pairs than one launch takes
    (65, 9, (5, 3, 7), torch.bfloat16, 4, 2),          # 210-byte pages; 130 pools, more than one launch takes
    (2, 7, (3, 1, 5), torch.uint8, 3, 3),
    (2, 6, (64, 8, 128), torch.float32, 3, 1),
]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("case", PAGES, ids=str)
def test_copy_kv_blocks(case, dev):
    layers, nb, page, dt, pairs, sources = case
    g = torch.Generator().manual_seed(1)
    pools = [torch.randint(0, 250, (nb, *page), generator=g).to(dt).to(dev) for _ in range(2 * layers)]
    ids = torch.randperm(nb, generator=g).tolist()
    src = [ids[i % sources] for i in range(pairs)]
    dst = ids[sources:sources + pairs]
    want = [t.clone() for t in pools]
    for t in want:
        for a, b in zip(src, dst):
            t[b] = t[a]
    serving.copy_kv_blocks(pools[:layers], pools[layers:], src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    copier = serving.KVBlockCopier(pools[:layers], [paddle.Tensor._wrap(t) for t in pools[layers:]])
    copier.copy([], [])
    copier.copy(tuple(src), dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copy_kv_blocks_refusals():
    k = [torch.arange(6.0).reshape(6, 1) for _ in range(2)]
    v = [t.clone() for t in k]
    c = serving.KVBlockCopier(k, v)
    bad = [([0], [6]), ([-1], [2]), ([6], [2]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0, 1], [2])]
    for s, d in bad:
        with pytest.raises(ValueError):
            c.copy(s, d)
        with pytest.raises(ValueError):
            N.native().kv_copy_check(s, d, 6)
    assert all(torch.equal(t, torch.arange(6.0).reshape(6, 1)) for t in k + v)
    N.native().kv_copy_check([0, 0, 5], [1, 2, 3], 6)
    for ks, vs in (([], []), (k, [t.double() for t in v]), (k, [t[:3] for t in v]), ([torch.zeros(4, 6).t()], []),
                   ([torch.zeros(1, 3).expand(4, 3)], []), ([torch.zeros(4)], [])):
        with pytest.raises(ValueError):
            serving.KVBlockCopier(ks, vs)


@pytest.mark.gpu
def test_copy_kv_blocks_gpu_placements():
    """Pages with gaps between them, pages past 2^31 bytes, another stream, a captured copy."""
    pool = torch.arange(8 * 40, device="cuda").reshape(8, 40).to(torch.int32)
    view = pool[:, 3:13]                                   # 40-byte pages at 4-byte addresses, 160 bytes apart
    want = pool.clone()
    want[5, 3:13] = want[2, 3:13]
    serving.copy_kv_blocks([view], [], [2], [5])
    assert torch.equal(pool, want)
    big = torch.zeros(5, 2 ** 30, dtype=torch.uint8, device="cuda")
    big[0] = 3
    big[0, -5:] = 9
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        serving.copy_kv_blocks([big], [], [0, 0], [4, 2])
    s.synchronize()
    assert torch.equal(big[4], big[0]) and torch.equal(big[2], big[0]) and not big[1].any() and not big[3].any()
    del big
    k, v = (torch.randn(6, 16, 2, 64, device="cuda") for _ in range(2))
    c = serving.KVBlockCopier([k], [v])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.copy([0, 1], [4, 5])
    for _ in range(3):
        k.normal_(), v.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(k[4:], k[:2]) and torch.equal(v[4:], v[:2])


# ============================================================================ sampling
def _token64(row, u, t, k, p, m):
    """One row by the definition: an explicit sorted list, 64 bits (Python floats and exact sums)."""
    row = [float("-inf") if x != x else x for x in row]
    top = max(row)
    if t == 0 or top == float("-inf"):
        return row.index(top)
    w = [1.0 if x == top else 0.0 if x == float("-inf") or top == float("inf") else math.exp((x - top) / t) for x in row]
    order = sorted(range(len(row)), key=lambda i: (-row[i], i))
    if k > 0:
        order = order[:k]
    if p < 1:
        z, kept, mass = math.fsum(w[i] for i in order), [], 0.0
        for i in order:
            if kept and not mass < p * z:
                break
            kept.append(i)
            mass = math.fsum([mass, w[i]])
        order = kept
    order = sorted(i for i in order if w[i] >= m)
    z, c = math.fsum(w[i] for i in order), 0.0
    order = [i for i in order if w[i] > 0]
    for i in order:
        c = math.fsum([c, w[i]])
        if c > u * z:
            return i
    return order[-1]


def _f32(v):
    return torch.tensor(v, dtype=torch.float32).item()


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_p=0.0),
            dict(top_p=0.5), dict(temperature=1.7, top_p=0.97), dict(min_p=0.2), dict(min_p=1.0),
            dict(temperature=0.8, top_k=20, top_p=0.7, min_p=0.01), dict(top_k=10 ** 9, top_p=1.0), dict(top_k=-1)]


def _check_sample(dev, dtype, B, V, setting, seed=0, coarse=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 3
    if coarse:
        x = x.round()          # many equal logits
    x[torch.rand(B, V, generator=g) < 0.1] = float("-inf")
    x[:, 0] = 0.0
    x = x.to(dtype)
    u = torch.rand(B, generator=g)
    u[0] = 0.0
    u[-1] = 1 - 2.0 ** -24
    got = serving.sample_tokens(x.to(dev), u.to(dev), **setting)
    s = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **{})
    s.update(setting)
    want = [_token64(x[b].double().tolist(), u[b].item(), _f32(s["temperature"]), s["top_k"], _f32(s["top_p"]),
                     _f32(s["min_p"])) for b in range(B)]
    assert got.dtype == torch.int64 and got.tolist() == want


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_sample_tokens_cpu(setting):
    _check_sample("cpu", torch.float32, 6, 97, setting)
    _check_sample("cpu", torch.bfloat16, 5, 513, setting, coarse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_sample_tokens_gpu(setting, dtype):
    for i, (B, V) in enumerate([(1, 1), (2, 2), (7, 97), (5, 513), (3, 4096), (4, 8193), (2, 20011)]):
        _check_sample("cuda", dtype, B, V, setting, seed=i)
        _check_sample("cuda", dtype, B, V, setting, seed=i, coarse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.01, 1.0, 8.0])
@pytest.mark.parametrize("V", [50257, 131072, 400000])
def test_sample_tokens_wide_rows_gpu(V, spread):
    """Long rows, flat and sharp, every kind of setting, against the CPU definition."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g) * spread
    u = torch.rand(8, generator=g)
    for s in (dict(), dict(top_p=0.9), dict(top_p=0.999), dict(top_k=50), dict(top_k=V // 2, top_p=0.6), dict(min_p=0.3),
              dict(temperature=0.5, top_k=3000, min_p=0.02)):
        for dt in (torch.float32, torch.bfloat16):
            xs = x.to(dt)
            want = serving.sample_tokens(xs, u, **s)
            assert torch.equal(serving.sample_tokens(xs.cuda(), u.cuda(), **s).cpu(), want), (s, dt)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sample_tokens_settings_per_row(dev):
    g = torch.Generator().manual_seed(5)
    B, V = 40, 300
    x = torch.randn(B, V, generator=g) * 2
    u = torch.rand(B, generator=g)
    t = torch.rand(B, generator=g) * 2
    t[::5] = 0
    t[1] = -1.0
    t[2] = float("nan")
    k = torch.randint(-2, 40, (B,), generator=g)
    k[7] = 2 ** 40
    p = torch.rand(B, generator=g) * 1.3
    p[8], p[9] = float("nan"), -0.5
    m = torch.rand(B, generator=g) * 0.2
    m[10], m[11] = float("nan"), 3.0
    got = serving.sample_tokens(x.to(dev), u.to(dev), t.to(dev), k.to(dev), p.to(dev), m.to(dev)).tolist()
    for b in range(B):
        tb = t[b].item() if t[b] > 0 else 0.0
        pb = 1.0 if p[b] != p[b] else p[b].item()
        mb = 0.0 if m[b] != m[b] else min(m[b].item(), 1.0)
        assert got[b] == _token64(x[b].double().tolist(), u[b].item(), tb, int(k[b]), pb, mb), b


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sample_tokens_odd_rows(dev):
    inf, nan = float("inf"), float("nan")
    rows = [([-inf] * 4, 0.9, 0), ([nan] * 4, 0.9, 0), ([nan, -inf, 2.0, nan], 0.99, 2), ([1.0, inf, 5.0, inf], 0.4, 1),
            ([1.0, inf, 5.0, inf], 0.6, 3), ([0.0, -0.0, 0.0, -0.0], 0.3, 1), ([0.0, -0.0, 0.0, -0.0], 0.5, 2),
            ([-3e38, -3e38, -inf, -3e38], 0.5, 1), ([3e38, -3e38, 1.0, 0.0], 0.9999, 0), ([0.0] * 4, 1.0, 3),
            ([0.0] * 4, inf, 3), ([0.0] * 4, nan, 0), ([0.0] * 4, -1.0, 0), ([0.0, 0.0, -inf, -inf], 1.0, 1)]
    x = torch.tensor([r[0] for r in rows], device=dev)
    u = torch.tensor([r[1] for r in rows], device=dev)
    assert serving.sample_tokens(x, u).tolist() == [r[2] for r in rows]
    # equal logits at the border: the lowest indexes are kept, whichever setting draws it
    flat = torch.zeros(4, 8, device=dev)
    u = torch.tensor([0.0, 0.26, 0.74, 0.999], device=dev)
    assert serving.sample_tokens(flat, u, top_k=3).tolist() == [0, 0, 2, 2]
    assert serving.sample_tokens(flat, u, top_p=0.5).tolist() == [0, 1, 2, 3]
    assert serving.sample_tokens(flat, u, top_k=4, top_p=0.5).tolist() == [0, 0, 1, 1]
    assert serving.sample_tokens(flat, u, temperature=0).tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sample_tokens_shares(dev):
    """u on an even grid draws every token in the share of its weight, to one in each direction."""
    n = 4000
    w = torch.tensor([0.4, 0.3, 0.2, 0.06, 0.04])
    x = w.log().repeat(n, 1).to(dev)
    u = ((torch.arange(n) + 0.5) / n).to(dev)
    got = torch.bincount(serving.sample_tokens(x, u), minlength=5).cpu()
    assert ((got - n * w).abs() <= 1).all()
    got = torch.bincount(serving.sample_tokens(x, u, top_p=0.85), minlength=5).cpu()
    assert ((got - n * torch.tensor([0.4, 0.3, 0.2, 0, 0]) / 0.9).abs() <= 1).all()
    got = torch.bincount(serving.sample_tokens(x, u, min_p=0.12), minlength=5).cpu()
    assert ((got - n * torch.tensor([0.4, 0.3, 0.2, 0.06, 0]) / 0.96).abs() <= 1).all()


@pytest.mark.gpu
def test_sample_tokens_views_streams_and_graphs_gpu():
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(16, 1200, generator=g).to(torch.bfloat16)
    u = torch.rand(16, generator=g)
    s = dict(temperature=0.9, top_k=40, top_p=0.9)
    for view in (lambda t: t[:, 1:1002], lambda t: t[::2, 3:700], lambda t: t.t()[:16, :16], lambda t: t[:, ::3]):
        v = view(wide)
        want = serving.sample_tokens(v, u[:v.shape[0]], **s)
        assert torch.equal(serving.sample_tokens(view(wide.cuda()), u[:v.shape[0]].cuda(), **s).cpu(), want)
    x, ud = wide.cuda(), u.cuda()
    out = torch.empty(16, dtype=torch.int64, device="cuda")
    serving.sample_tokens(x, ud, **s, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serving.sample_tokens(x, ud, **s)
    for i in range(4):
        x.copy_(torch.randn(16, 1200, generator=g).to(torch.bfloat16))
        ud.copy_(torch.rand(16, generator=g))
        graph.replay()
        eager = serving.sample_tokens(x, ud, **s)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(got.cpu(), serving.sample_tokens(x.cpu(), ud.cpu(), **s))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = serving.sample_tokens(x, ud, **s)
    st.synchronize()
    assert torch.equal(other, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("V,shift", [(1000, 0.0), (33000, 500.0), (70001, -3e4)])
def test_sample_tokens_min_p_at_every_temperature_gpu(V, shift):
    """min-p alone, temperatures and floors from the smallest to the largest, logits far from zero: as in 64 bits on the CPU."""
    t, m = torch.meshgrid(torch.tensor([1e-30, 1e-3, 0.7, 50.0, 1e30, float("inf")]),
                          torch.tensor([1e-38, 1e-6, 0.05, 0.5, 1.0, 2.0, float("nan")]), indexing="ij")
    t, m = t.flatten(), m.flatten()
    g = torch.Generator().manual_seed(V)
    x = torch.randn(len(t), V, generator=g) * 4 + shift
    x[:, 7] = x.amax(1)
    x[::5, ::3] = float("-inf")
    u = torch.rand(len(t), generator=g)
    want = serving.sample_tokens(x, u, temperature=t, min_p=m)
    got = serving.sample_tokens(x.cuda(), u.cuda(), temperature=t.cuda(), min_p=m.cuda())
    assert torch.equal(got.cpu(), want)


def test_sample_tokens_refusals():
    x, u = torch.zeros(3, 5), torch.zeros(3)
    f = serving.sample_tokens
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_p=1.5),
               dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=-1.0), dict(top_k=2.5), dict(top_k=-7), dict(top_k="3"), dict(top_k=float("inf")),
               dict(temperature=torch.zeros(2)), dict(top_k=torch.zeros(3, 1, dtype=torch.int32)),
               dict(out=torch.zeros(3)), dict(out=torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            f(x, u, **kw)
    for a, b in ((x[0], u), (x[:, :0], u), (x.long(), u), (x, u[:2]), (x, u.double())):
        with pytest.raises(ValueError):
            f(a, b)
    with pytest.raises(TypeError):
        f(x, u, top_k=torch.zeros(3))
    assert f(x[:0], u[:0]).shape == (0,)
    t = f(paddle.Tensor._wrap(x), paddle.Tensor._wrap(u))
    assert isinstance(t, paddle.Tensor) and t._t.tolist() == [0, 0, 0]


# ============================================================================ together
def _cache(dev, **kw):
    d = dict(num_layers=2, num_blocks=12, block_size=4, num_kv_heads=1, head_dim=8, max_batch=5, max_seq_len=16,
             dtype=torch.float32, device=torch.device(dev))
    d.update(kw)
    return serving.PagedKVCache(**d)


def _rows(c, slot, n, layer=0):
    j = torch.arange(n, device=c.k[0].device)
    return c.k[layer][c.block_table[slot].long()[j // c.block_size], j % c.block_size]


def _put(c, slot, start, n, value):
    dev = c.k[0].device
    rows = (torch.arange(start, start + n, device=dev).float() + value)[:, None, None].expand(n, 1, 8).contiguous()
    for k, v in zip(c.k, c.v):
        serving.write_kv(rows, -rows, k, v, torch.full((n,), slot, device=dev), torch.arange(start, start + n, device=dev),
                         c.block_table)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_paged_cache_fork_truncate_compact(dev):
    c = _cache(dev)
    c.allocate(0, 11)
    _put(c, 0, 0, 10, 100)
    c.seq_lens[0] = 10
    c.fork(0, [2, 3])
    assert c.num_free_blocks == 12 - 3 - 2 and c.seq_lens.tolist() == [10, 0, 10, 10, 0]
    want = _rows(c, 0, 10).clone()
    for s in (2, 3):
        assert torch.equal(_rows(c, s, 10), want) and torch.equal(_rows(c, s, 10, 1), want)
        c.allocate(s, 12)
        _put(c, s, 10, 2, 1000 * s)
    _put(c, 0, 10, 1, 500)
    assert _rows(c, 0, 11)[10, 0, 0] == 510 and _rows(c, 2, 12)[10, 0, 0] == 2010 and _rows(c, 3, 12)[11, 0, 0] == 3011
    assert all(torch.equal(_rows(c, s, 10), want) for s in (0, 2, 3))
    # back into a shared page: it becomes the sequence's own before it is written
    c.truncate(2, 6)
    _put(c, 2, 6, 2, 7000)
    assert torch.equal(_rows(c, 0, 10), want) and torch.equal(_rows(c, 3, 10), want)
    assert _rows(c, 2, 8)[6, 0, 0] == 7006 and torch.equal(_rows(c, 2, 6), want[:6]) and int(c.seq_lens[2]) == 6
    c.free(0)
    before = {s: _rows(c, s, n).clone() for s, n in ((2, 8), (3, 12))}
    used = 12 - c.num_free_blocks
    c.compact()
    assert sorted({b for s in (2, 3) for b in c._owned[s]}) == list(range(used)) and 12 - c.num_free_blocks == used
    assert c.compact() == 0
    for s, n in ((2, 8), (3, 12)):
        assert torch.equal(_rows(c, s, n), before[s]) and torch.equal(_rows(c, s, n, 1), before[s])
    c.free(2), c.free(3)
    assert c.num_free_blocks == 12 and sorted(c._free) == list(range(12)) and not any(c._holders)
    c.truncate(1, 0)
    c.fork(1, [0])
    assert c.num_free_blocks == 12


def test_paged_cache_refusals():
    c = _cache("cpu")
    c.allocate(0, 10)
    c.allocate(1, 16)
    for f in (lambda: c.fork(0, [1], 4), lambda: c.fork(0, [2, 2], 4), lambda: c.fork(0, [0], 4), lambda: c.fork(0, [2], 13),
              lambda: c.fork(0, [2], -1), lambda: c.truncate(0, 13), lambda: c.truncate(4, 1)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: c.fork(0, [5], 4), lambda: c.fork(-1, [2], 4), lambda: c.truncate(9, 0), lambda: c.allocate(2, 17)):
        with pytest.raises(IndexError):
            f()
    c.free(2)
    c.allocate(2, 16)
    state = (list(c._free), {k: list(v) for k, v in c._owned.items()}, list(c._holders))
    with pytest.raises(RuntimeError):
        c.fork(0, [3, 4], 9)     # two pages wanted, one free
    assert state == (c._free, c._owned, c._holders)


def _llama(dev, **kw):
    from paddle2_amd.models import LlamaConfig, LlamaForCausalLM

    paddle.seed(3)
    cfg = LlamaConfig.tiny(num_attention_heads=4, num_key_value_heads=2, dtype="bfloat16" if dev == "cuda" else "float32", **kw)
    m = LlamaForCausalLM(cfg)
    if dev == "cuda":
        paddle.set_device("gpu:0")
        m.to(device="gpu:0")
    m.eval()
    return m


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_extend_is_prefill_in_pieces(dev):
    """Chunks of a ragged batch give the whole prompt's cache rows and last logits."""
    from paddle2_amd.serving import LlamaGenerator

    m = _llama(dev)
    prompts = [[(7 * i + 3) % 500 for i in range(41)], [9, 8, 7], [(5 * i) % 400 for i in range(20)]]
    a = LlamaGenerator(m, max_batch=3, max_seq_len=64, block_size=8, use_graph=False)
    b = LlamaGenerator(m, max_batch=3, max_seq_len=64, block_size=8, use_graph=False)
    whole = a.prefill_batch([0, 1, 2], prompts)
    parts = b.prefill_chunks([0, 1, 2], prompts, 13)
    tol = dict(atol=3e-2, rtol=3e-2) if dev == "cuda" else dict(atol=1e-4, rtol=1e-4)
    torch.testing.assert_close(parts.float(), whole.float(), **tol)
    assert a.cache.seq_lens.tolist() == b.cache.seq_lens.tolist() == [41, 3, 20]
    for x, y in zip(a.cache.k + a.cache.v, b.cache.k + b.cache.v):
        for s, n in ((0, 41), (1, 3), (2, 20)):
            j = torch.arange(n, device=x.device)
            torch.testing.assert_close(x[a.cache.block_table[s].long()[j // 8], j % 8].float(),
                                       y[b.cache.block_table[s].long()[j // 8], j % 8].float(), **tol)
    with pytest.raises(ValueError):
        b.extend([0, 0], [[1], [2]])
    with pytest.raises(ValueError):
        b.extend([0], [[]])
    with pytest.raises(ValueError):
        b.prefill_chunks([0], [[1]], 0)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_generate_with_shared_prompts_and_fused_sampling(dev):
    from paddle2_amd.serving import LlamaGenerator

    m = _llama(dev)
    prompts = [[1, 5, 9, 3, 11, 4, 8, 2, 6], [7, 2, 8]]
    gen = LlamaGenerator(m, max_batch=6, max_seq_len=64, block_size=8, use_graph=dev == "cuda")
    plain = gen.generate(prompts, 5)
    # greedy continuations of one prompt are the same, whichever sampler, in pieces or not
    again = gen.generate(prompts, 5, num_return_sequences=3)
    fused = gen.generate(prompts, 5, sampler="fused", chunk_size=4 if dev == "cpu" else None)
    first = 1 if dev == "cuda" else 5     # bf16: a batch of another size may flip a near tie later on
    for i in range(6):
        assert again[i][:first] == plain[i // 3][:first]
    assert [f[:first] for f in fused] == [p[:first] for p in plain]
    kw = dict(temperature=0.9, top_k=30, min_p=0.02, seed=4, num_return_sequences=3)
    one, two = gen.generate(prompts, 6, **kw), gen.generate(prompts, 6, **kw)
    assert one == two and all(len(o) == 6 and all(0 <= t < 512 for t in o) for o in one)
    mixed = gen.generate(prompts, 5, temperature=[0.0, 1.0], top_p=[1.0, 0.9], seed=1)
    assert mixed[0][:first] == plain[0][:first]
    assert gen.cache.num_free_blocks == len(gen.cache._holders)
    for bad in (dict(sampler="multinomial", min_p=0.1), dict(sampler="beam"), dict(temperature=[1.0])):
        with pytest.raises(ValueError):
            gen.generate(prompts, 3, **bad)


def test_shared_pages_are_not_written():
    """A prompt, a chunk or a whole generation over a slot that shares the pages it would write is refused, with nothing
    changed; pools that were added to a cache are copied too."""
    from paddle2_amd.serving import LlamaGenerator

    gen = LlamaGenerator(_llama("cpu"), max_batch=3, max_seq_len=64, block_size=8, use_graph=False)
    gen.prefill_chunks([0], [list(range(1, 22))], 8)
    gen.cache.fork(0, [1])
    pools = [t.clone() for t in gen.cache.k + gen.cache.v]
    for f in (lambda: gen.extend([1], [[5]], held=[15]), lambda: gen.prefill(1, torch.tensor([3, 4])),
              lambda: gen.prefill_batch([2, 0], [[1], [2]]), lambda: gen.generate([[1, 2]], 2)):
        with pytest.raises(ValueError, match="shares pages"):
            f()
    assert all(torch.equal(a, b) for a, b in zip(pools, gen.cache.k + gen.cache.v))
    gen.cache.truncate(1, 15)
    gen.extend([1], [[5]], held=[15])
    gen.extend([0], [[5]], held=[16])    # behind the shared pages
    gen.cache.free(1), gen.cache.free(0)
    assert len(gen.generate([[1, 2]], 2)[0]) == 2

    c = _cache("cpu")
    c.copy_blocks([0], [1])
    c.k.append(torch.arange(12.0).repeat_interleave(c.k[0][0].numel()).view_as(c.k[0]).to(c.k[0].dtype))
    c.v.append(c.k[-1].clone())
    c.copy_blocks([3], [5])
    assert (c.k[-1][5] == 3).all() and (c.v[-1][5] == 3).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_drafted_tokens_checked_and_rejected(dev):
    """A forked sequence takes drafted tokens in one extend, is truncated to the accepted ones, and goes on as one that
    never saw the others."""
    from paddle2_amd.serving import LlamaGenerator

    m = _llama(dev)
    gen = LlamaGenerator(m, max_batch=3, max_seq_len=64, block_size=8, use_graph=False)
    prompt = [(11 * i + 1) % 300 for i in range(21)]
    gen.prefill_chunks([0], [prompt], 8)
    gen.cache.fork(0, [1, 2])
    gen.extend([1], [[5, 6, 7, 8]])
    gen.cache.truncate(1, 23)            # 5 and 6 are kept
    a = gen.extend([1], [[9, 10]])
    b = gen.extend([2], [[5, 6, 9, 10]])
    assert gen.cache.seq_lens.tolist() == [21, 25, 25]
    tol = dict(atol=3e-2, rtol=3e-2) if dev == "cuda" else dict(atol=1e-4, rtol=1e-4)
    torch.testing.assert_close(a.float(), b.float(), **tol)
    gen.cache.compact()
    u = torch.full((1,), 0.37, device=a.device)
    tok = serving.sample_tokens(gen.extend([1], [[3]]), u, 0.8, 20, 0.9)
    assert 0 <= int(tok) < 512


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_block_multihead_attention_several_new_tokens(dev):
    """Sequences that bring several tokens behind cached ones, beside a decoding one and a prompt."""
    dt = torch.float32 if dev == "cpu" else torch.bfloat16
    Hq, Hk, D, bs = 4, 2, 64, 16
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn(12, Hk, bs, D, generator=g).to(dev, dt) for _ in range(2))
    table = torch.arange(12, dtype=torch.int32).reshape(4, 3).to(dev)
    enc, dec, now = [0, 0, 6, 0], [30, 17, 0, 5], [3, 1, 6, 9]
    cu = torch.tensor([0, 3, 4, 10, 19], dtype=torch.int32)
    qkv = torch.randn(19, (Hq + 2 * Hk) * D, generator=g).to(dev, dt)
    W = paddle.Tensor._wrap
    i32 = lambda v: W(torch.tensor(v, dtype=torch.int32, device=dev))  # noqa: E731
    out = serving.block_multihead_attention(W(qkv), W(kc), W(vc), i32(enc), i32(dec), i32(now), None, None,
                                            W(cu.to(dev)), W(cu.to(dev)), W(table), block_size=bs)[0]._t
    q = qkv.reshape(19, Hq + 2 * Hk, D)[:, :Hq]
    lens = torch.tensor([d + n for d, n in zip(dec, now)], dtype=torch.int32)
    o, a, big = _attn64(q, kc, vc, cu, lens, table, layout="paddle_block")
    err = (out.reshape(19, Hq, D).double().cpu() - o).abs()
    assert (err[[0, 1, 2] + list(range(10, 19))] <= _tolerance(dt, D, o, a, big)[[0, 1, 2] + list(range(10, 19))]).all()
    assert (err <= 0.05).all()
