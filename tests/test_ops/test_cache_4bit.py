"""4-bit caches: the numbers and their layout, appending to pools (in 4 bits and in the activations' type), and attention over 4 bits.

Codes are those of the exact keys and values: they have to be equal. Queries, and keys of other pools, are rounded once (``eps / 2``) after
float32 arithmetic of at most 32 roundings of the row's largest value (as in test_norm_rope.py). Attention: the output is rounded once, 2^-8 of
it; each weight is rounded to bfloat16, 2^-8 of sum p |v|; a score's float32 error, D + 2 roundings of scale * sum |q k|, moves a weight by as
much of itself, and so does the sum over L keys with at most L 2^-24."""

import math

import pytest
import torch

from colossalai_amd.inference.kv_cache import KVCacheManager  # noqa: F401  (pages are addressed as there)
from colossalai_amd.ops import build_rope_table, kv4_pool, kv4_read, paged_attention_4bit, paged_kv_append
from colossalai_amd.ops.cache_4bit import _tiles, kv4_unpack
from colossalai_amd.ops.ragged import RaggedBatch

gpu = pytest.mark.gpu
EACH = ["cpu", pytest.param("cuda", marks=gpu)]
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _nearest(x):
    """The numbers of a 4-bit cache for x [.., D]: by trying every power of two and every number."""
    x = x.double().unflatten(-1, (-1, 32))
    powers = torch.exp2(torch.arange(-126, 128, dtype=torch.float64, device=x.device))
    most = x.abs().amax(-1, keepdim=True)
    fit = (6 * powers >= most).int().argmax(-1)  # the first that fits
    unit = powers[fit].unsqueeze(-1)
    a = x.abs() / unit
    away = (a.unsqueeze(-1) - GRID.to(x.device)).abs()
    best = away == away.amin(-1, keepdim=True)
    even = best & (torch.arange(8, device=x.device) % 2 == 0)
    pick = torch.where(best.sum(-1) > 1, even.int().argmax(-1), best.int().argmax(-1))
    out = torch.sign(x) * GRID.to(x.device)[pick] * unit
    return torch.where((most < math.inf), out, math.nan).flatten(-2)


def _turned(x, w, table, at, eps):
    x, half = x.double(), x.shape[-1] // 2
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = table.double()[at.long()][:, None].chunk(2, -1)
    return torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("device", EACH)
def test_layout(D, device):
    """Each code and scale byte where the layout says, read one by one."""
    pool = torch.randint(0, 250, (2, 3, 32 * 17 * D // 32), generator=torch.Generator().manual_seed(D)).byte()  # 6 * 2^(249 - 127) is finite
    keys, values = (kv4_unpack(pool, D, v) for v in (False, True))
    assert keys.shape == values.shape == (2, 32, 3, D)
    read = kv4_read(pool.to(device), pool.to(device), torch.arange(64, device=device).int(), D)
    g = torch.Generator().manual_seed(7)
    for _ in range(200):
        p, t, h, c = (int(torch.randint(0, n, (), generator=g)) for n in (2, 32, 3, D))
        tile = pool[p, h].view(-1, 17 * D // 2)[t // 16]
        places = (((t % 16) * (D // 2) + c // 2, 8 * D + (t % 16) * (D // 32) + c // 32),
                  (((t % 16 // 4 * 16 + c // (D // 16)) * 4 + t % 4) * (D // 32) + c % (D // 16) // 2, 8 * D + c // 32 * 16 + t % 16))
        for got, back, (code_at, scale_at) in zip((keys, values), read, places):
            code, byte = int(tile[code_at]) >> 4 * (c % 2) & 15, int(tile[scale_at])
            want = float(GRID[code & 7]) * (-1 if code & 8 else 1) * (2.0 ** (byte - 127) if byte else 0.0)
            if byte:
                assert float(got[p, t, h, c]) == want
                assert abs(want) < 2.0 ** -126 or float(back[p * 32 + t, h, c]) == want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("device", EACH)
def test_borders_and_extremes(D, dtype, device):
    """Values next to the borders of codes and scales, ties, zeros, the smallest and largest numbers, and what is not finite; a
    position of 0, so that keys are turned by nothing."""
    N, G = 40, 2
    x = torch.randn(N, G, D, generator=torch.Generator().manual_seed(1))
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 4.0, 3.0])
    x[0, 0, :32] = 6.0
    x[0, 0, 1:11] = steps
    x[0, 1, :32] = 0.0
    x[1, 0, :10] = -steps * 2.0 ** 100
    x[1, 0, 10:32] = 6.0 * 2.0 ** 100
    x[1, 1, :32] *= 2.0 ** -125
    x[2, 0, :32] = 2.0 ** -130
    x[2, 1, 3] = 2.9e38  # the largest numbers are 3 and -3 times 2^126: 3.5 times it and more become infinite
    x[3, 0, :32] = 0.0
    x[3, 0, 5] = 6.0 * (1 + 2.0 ** -7)  # just over a scale's border
    x[3, 1, 5], x[3, 1, 37] = math.inf, math.nan
    x[4, 0, 0] = -math.inf
    x = x.to(device, dtype)
    kpool, vpool = (kv4_pool(4, 16, G, D, device) for _ in range(2))
    rows = torch.randperm(64, generator=torch.Generator().manual_seed(2))[:N].int().to(device)
    table = build_rope_table(4, D, 1e4, device)
    q = torch.zeros(N, 4, D, device=device, dtype=dtype)
    paged_kv_append(q, x, x, kpool, vpool, rows, torch.zeros_like(rows), table)
    want = _nearest(x)
    normal = want.abs().nan_to_num(1.0) >= 2.0 ** -126  # below, what a conversion gives is the arithmetic's affair
    # a NaN or infinity beside a finite channel: turned by position 0 it meets 0 * inf in its pair
    bad = ~x.isfinite()
    half = D // 2
    paired = bad | torch.cat([bad[..., half:], bad[..., :half]], -1)
    want_k = torch.where(paired.unflatten(-1, (-1, 32)).any(-1, keepdim=True).expand(N, G, D // 32, 32).flatten(-2), math.nan, want)
    for got, w in zip(kv4_read(kpool, vpool, rows, D), (want_k, want)):
        assert torch.equal(got.isnan(), w.isnan())
        assert torch.equal(got.double()[normal & ~w.isnan()], w[normal & ~w.isnan()])
        assert (got.double()[~normal & ~w.isnan()].abs() <= 2.0 ** -126).all()


def _append_case(N, H, G, D, page, dtype, four, norm, wide, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(N, H + 2 * G, D, generator=g) * torch.exp(torch.randn(N, 1, 1, generator=g))).to(device, dtype)
    q, k, v = qkv.view(N, -1, D).split([H, G, G], 1)
    ws = [(1 + 0.3 * torch.randn(D, generator=g)).to(device, torch.float32 if wide else dtype) for _ in range(2)] if norm else [None] * 2
    pages = N // page + 3
    rows = torch.randperm(pages * page, generator=g)[:N].int().to(device)
    at = torch.randint(0, 300, (N,), generator=g).int().to(device)
    if four:
        pools = [torch.randint(0, 256, (pages, G, page * 17 * D // 32), generator=g).byte().to(device) for _ in range(2)]
    else:
        pools = [torch.randn(pages, page, G, D, generator=g).to(device, dtype) for _ in range(2)]
    return q, k, v, pools, rows, at, ws


def _bits(x):
    return x.contiguous().view({2: torch.int16, 4: torch.int32}[x.element_size()])


def _check_append(q, k, v, pools, rows, at, ws, table, eps=1e-6):
    D, four = q.shape[-1], pools[0].dtype == torch.uint8
    whole = [kv4_unpack(p, D, i == 1) if four else p.clone() for i, p in enumerate(pools)]
    whole = [p.clone().flatten(0, 1) for p in whole]
    out = paged_kv_append(q, k, v, *pools, rows, at, table, *ws, eps=eps)
    half = torch.finfo(q.dtype).eps / 2
    size = lambda y: half * y.abs() + 2.0 ** -18 * 1.42 * y.abs().amax(-1, keepdim=True)  # noqa: E731
    want = _turned(q, ws[0], table, at, eps)
    assert out.dtype == q.dtype and out.is_contiguous() and ((out.double() - want).abs() <= size(want)).all()
    key = _turned(k, ws[1], table, at, eps)
    kept = (rows >= 0) & (rows < whole[0].shape[0])
    into = rows[kept].long()
    others = torch.ones(whole[0].shape[0], dtype=torch.bool, device=q.device)
    others[into] = False
    for i, (p, w) in enumerate(zip(pools, whole)):
        now = (kv4_unpack(p, D, i == 1) if four else p).flatten(0, 1)
        assert torch.equal(_bits(now[others].nan_to_num(7.0)), _bits(w[others].nan_to_num(7.0))), "a row that is nobody's was written"
        if four:
            assert torch.equal(now[into].double(), _nearest(key if i == 0 else v)[kept])
        elif i == 0:
            assert ((now[into].double() - key[kept]).abs() <= size(key)[kept]).all()
        else:
            assert torch.equal(now[into], v[kept])
    return out


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("N,H,G,D,page,four,norm,wide", [
    (1, 1, 1, 64, 16, True, True, False), (3, 7, 1, 128, 16, True, True, True), (50, 8, 2, 128, 64, True, False, False),
    (333, 6, 2, 64, 32, True, True, False), (129, 4, 4, 256, 16, True, True, True), (2500, 3, 1, 128, 128, True, True, False),
    (1, 4, 2, 16, 1, False, True, False), (77, 5, 5, 80, 8, False, True, True), (400, 28, 4, 128, 16, False, False, False),
    (33, 2, 1, 512, 4, False, True, False), (20, 3, 3, 256, 2, False, True, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append(N, H, G, D, page, four, norm, wide, dtype, device):
    case = _append_case(N, H, G, D, page, dtype, four, norm, wide, device)
    _check_append(*case, build_rope_table(300, D, 1e4, device))


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("four", [True, False])
def test_append_padding_strides_and_positions(four, device):
    """Padding tokens and rows behind the pool are not written; heads that lie apart; positions that the table does not have."""
    q, k, v, pools, rows, at, ws = _append_case(40, 4, 2, 64, 16, torch.bfloat16, four, True, False, device)
    table = build_rope_table(300, 64, 1e4, device)
    rows[3], rows[7], rows[11] = -1, pools[0].shape[0] * 16, 2 ** 31 - 1
    mine = [p.clone() for p in pools]
    want = _check_append(q, k, v, mine, rows, at, ws, table)
    for lead in (8, 3):
        room = torch.zeros(40, lead + 3 * 64 * 8, device=device, dtype=torch.bfloat16)
        views = []
        for i, t in enumerate((q, k, v)):
            view = room[:, lead + i * 64 * 8: lead + i * 64 * 8 + t.shape[1] * 64].view(40, -1, 64)
            view.copy_(t)
            views.append(view)
        again = [p.clone() for p in pools]
        assert torch.equal(paged_kv_append(*views, *again, rows, at, table, *ws), want)
        assert all(torch.equal(a, b) for a, b in zip(again, mine))
    at[0], at[1] = 300, -1
    out = paged_kv_append(q, k, v, *pools, rows, at, table, *ws)
    assert out[:2].isnan().all() and torch.equal(out[2:], want[2:])
    if four:
        read = kv4_read(*pools, rows, 64)
        assert read[0][:2].isnan().all() and not read[1][:2].isnan().any()
        assert all(t[[3, 7, 11]].isnan().all() for t in read)
    none = [t[:0] for t in (q, k, v)]
    assert paged_kv_append(*none, *pools, rows[:0], at[:0], table, *ws).shape == (0, 4, 64)


def _batch(counts, starts, page, device, seed=0):
    need = [-(-(a + b) // page) for a, b in zip(counts, starts)]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at: at + n])
        at += n
    return RaggedBatch.build(counts, starts, list(range(len(counts))), device, tables, page), tables, sum(need) + 2


def _pools(tables, ends, pages, page, G, D, device, first=None):
    """Random codes; what no sequence holds (and what a window has left behind) has scales of 255 and large codes."""
    g = torch.Generator().manual_seed(pages)
    out = []
    for values in (False, True):
        pool = torch.randint(0, 256, (pages, G, page * 17 * D // 32), generator=g).byte()
        scales = _tiles(pool, D, values)[1]
        scales.copy_(torch.randint(124, 129, scales.shape, generator=g).byte())
        by_token = scales.transpose(-1, -2) if values else scales  # [pages, heads, tiles, 16, D / 32]
        held = torch.zeros(pages, page, dtype=torch.bool)
        for i, (t, end) in enumerate(zip(tables, ends)):
            for p in range(0 if first is None else first[i], end):
                held[t[p // page], p % page] = True
        by_token.masked_fill_(~held.view(pages, 1, page // 16, 16, 1), 255)
        out.append(pool.to(device))
    return out


def _check_attention(counts, starts, H, G, D, page, window=0, device="cuda", scale=None, spread=1.0):
    scale = D ** -0.5 if scale is None else scale
    batch, tables, pages = _batch(counts, starts, page, device)
    ends = [a + b for a, b in zip(counts, starts)]
    first = [max(0, s - window + 1) for s in starts] if window else None
    kpool, vpool = _pools(tables, ends, pages, page, G, D, device, first)
    q = (spread * torch.randn(sum(counts), H, D, generator=torch.Generator().manual_seed(5))).to(device, torch.bfloat16)
    got = paged_attention_4bit(q, kpool, vpool, batch, scale, window).double()
    assert got.shape == q.shape
    k, v = (kv4_unpack(p, D, x).double() for p, x in ((kpool, False), (vpool, True)))
    at = 0
    for n, s, end, t in zip(counts, starts, ends, tables):
        t = torch.tensor(t, device=device)
        kk, vv = (x[t].flatten(0, 1)[:end].nan_to_num(0.0).repeat_interleave(H // G, 1).transpose(0, 1) for x in (k, v))
        i, j = torch.arange(s, end, device=device)[:, None], torch.arange(end, device=device)[None]
        see = (j <= i) & ((i - j < window) | (window == 0))
        qq = q[at: at + n].double().transpose(0, 1)
        score = (qq @ kk.transpose(1, 2)) * scale
        size = float(((qq.abs() @ kk.abs().transpose(1, 2)) * abs(scale)).amax())
        p = torch.softmax(score.masked_fill(~see, -math.inf), -1)
        want, near = p @ vv, p @ vv.abs()
        slack = 2.0 ** -8 + 2 * (D + 2) * 2.0 ** -24 * size + 2 * end * 2.0 ** -24
        # float32 has no weights under 2^-126 (scores that are 87 and more behind): each of up to `end` keys may lose as much of its value
        least = 2.0 ** -126 * end * float(vv.abs().amax())
        off = (got[at: at + n].transpose(0, 1) - want).abs() - 2.0 ** -8 * want.abs() - slack * near - least
        assert (off <= 0).all(), f"{off.max():.2e} over the bound"
        at += n


DECODE = [
    ([1], [0], 1, 1, 64, 16), ([1], [0], 16, 2, 128, 64), ([1], [15], 4, 4, 256, 16), ([1], [16], 3, 1, 64, 32), ([1] * 3, [31, 32, 33], 7, 1, 128, 16),
    ([1] * 5, [0, 4999, 63, 1024, 2047], 8, 2, 128, 16), ([1] * 2, [9000, 3], 28, 4, 128, 64), ([1], [20011], 8, 1, 64, 16), ([1] * 4, [700, 3000, 1, 40], 20, 1, 128, 32),
    ([1] * 3, [1500, 2, 5000], 40, 2, 256, 64), ([1] * 2, [3000, 7], 130, 1, 64, 16), ([1] * 70, list(range(0, 1400, 20)), 4, 2, 64, 16)]
PORTIONS = [
    ([2], [0], 4, 2, 64, 16), ([16], [0], 1, 1, 128, 16), ([17, 1, 5], [3, 100, 0], 4, 2, 128, 16), ([33, 1, 96, 65], [0, 130, 31, 64], 8, 2, 128, 16),
    ([200], [1000], 7, 1, 64, 32), ([3, 64], [5000, 10], 6, 2, 256, 64), ([300, 40], [0, 77], 20, 1, 128, 16), ([2, 2, 1], [40, 3000, 6], 40, 2, 64, 16),
    ([513], [0], 12, 4, 256, 128), ([37, 1, 2], [100, 300, 20], 70, 1, 128, 16), ([9], [500], 260, 2, 64, 32), ([5], [60], 130, 1, 256, 16),
    ([95, 96, 24, 1], [10, 0, 2000, 50], 4, 4, 128, 16), ([40] * 9, [3000] * 9, 4, 1, 64, 64), ([4, 4, 4], [10, 200, 4000], 4, 1, 128, 16)]


@gpu
@pytest.mark.parametrize("counts,starts,H,G,D,page", DECODE + PORTIONS)
@pytest.mark.parametrize("window", [0, 1, 100])
def test_attention(counts, starts, H, G, D, page, window):
    _check_attention(counts, starts, H, G, D, page, window)


@pytest.mark.parametrize("counts,starts,H,G,D,page,window", [([1], [0], 2, 1, 64, 16, 0), ([5, 1], [30, 17], 4, 2, 128, 16, 0), ([9], [40], 3, 3, 64, 32, 12)])
def test_attention_on_the_cpu(counts, starts, H, G, D, page, window):
    _check_attention(counts, starts, H, G, D, page, window, "cpu")


@gpu
@pytest.mark.parametrize("scale,spread", [(-0.3, 1.0), (0.0, 1.0), (1.0, 20.0)])
def test_attention_scales(scale, spread):
    """Negative, zero and large scores: a weight's error grows with the scores' size, as the bound does."""
    _check_attention([1, 30, 1], [2500, 100, 40], 8, 2, 128, 16, scale=scale, spread=spread)


@gpu
def test_not_finite_values_stay_with_the_tokens_that_see_them():
    """In a portion, tokens ahead of a key or value that is not finite do not show it, those from it on do."""
    page, D, G, H, n = 16, 128, 2, 4, 50
    batch, tables, pages = _batch([n], [20], page, "cuda")
    clean = _pools(tables, [70], pages, page, G, D, "cuda")
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(5)).to("cuda", torch.bfloat16)
    want = paged_attention_4bit(q, *clean, batch, 0.1)
    for values in (False, True):
        for where in (20, 37, 48, 69):
            pools = [p.clone() for p in clean]
            scales = _tiles(pools[values], D, values)[1]
            by_token = scales.transpose(-1, -2) if values else scales
            by_token[tables[0][where // page], 1, 0, where % page, 2] = 255
            got = paged_attention_4bit(q, *pools, batch, 0.1)
            assert torch.equal(got[:, :2], want[:, :2])
            assert torch.equal(got[: where - 20], want[: where - 20])
            assert got[where - 20:, 2:].isnan().any(-1).all()


@gpu
def test_pages_that_the_pool_does_not_have():
    """They give NaN to the tokens that see them, and nothing else."""
    batch, tables, pages = _batch([1, 1, 40], [100, 90, 10], 16, "cuda")
    pools = _pools(tables, [101, 91, 50], pages, 16, 2, 64, "cuda")
    q = torch.randn(42, 4, 64, device="cuda").bfloat16()
    want = paged_attention_4bit(q, *pools, batch, 0.1)
    batch.block_tables[0, 2], batch.block_tables[2, 2] = pages, -5
    got = paged_attention_4bit(q, *pools, batch, 0.1)
    assert got[0].isnan().all() and torch.equal(got[1], want[1]) and torch.equal(got[2:24], want[2:24]) and got[24:].isnan().all()


@gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes, its last pages in use."""
    page, G, D, H = 256, 8, 256, 8
    size = G * page * 17 * D // 32
    pages = 2 ** 32 // size + 40
    kpool, vpool = (torch.zeros(pages, G, page * 17 * D // 32, dtype=torch.uint8, device="cuda") for _ in range(2))
    tables = [[pages - 1, 0, pages - 2], [3, pages - 3]]
    batch = RaggedBatch.build([700, 260], [0, 0], [0, 1], "cuda", tables, page)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(960, H + 2 * G, D, device="cuda", generator=g).bfloat16()
    table = build_rope_table(1024, D, 1e4, "cuda")
    q = paged_kv_append(x[:, :H], x[:, H: H + G], x[:, H + G:], kpool, vpool, batch.kv_rows, batch.positions, table)
    got = paged_attention_4bit(q, kpool, vpool, batch, D ** -0.5)
    pick = torch.tensor([pages - 1, 0, pages - 2, 3, pages - 3], device="cuda")
    small = RaggedBatch.build([700, 260], [0, 0], [0, 1], "cuda", [[0, 1, 2], [3, 4]], page)
    assert torch.equal(got, paged_attention_4bit(q, kpool[pick].contiguous(), vpool[pick].contiguous(), small, D ** -0.5))
    assert got.isfinite().all()


@gpu
def test_together_on_another_stream_and_in_a_captured_graph():
    """A step as an engine makes it, append then attend, on a stream of its own and replayed with new inputs."""
    H, G, D, page = 8, 2, 128, 16
    counts, starts = [1, 1, 30, 1], [700, 3, 50, 4000]
    batch, tables, pages = _batch(counts, starts, page, "cuda")
    start = _pools(tables, [a + b for a, b in zip(counts, starts)], pages, page, G, D, "cuda")
    ws = [torch.rand(D, device="cuda").bfloat16() + 0.5 for _ in range(2)]
    table = build_rope_table(4096, D, 1e4, "cuda")
    x = torch.randn(33, H + 2 * G, D, device="cuda").bfloat16()
    pools = [p.clone() for p in start]

    def step(pools):
        q, k, v = x.split([H, G, G], 1)
        q = paged_kv_append(q, k, v, *pools, batch.kv_rows, batch.positions, table, *ws)
        return paged_attention_4bit(q, *pools, batch, D ** -0.5)

    want = step(pools)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [p.clone() for p in start]
        got = step(other)
    side.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(other, pools))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for graph in graphs:  # two graphs, replayed in turn
        with torch.cuda.graph(graph):
            held.append(step(pools))
    for turn in range(4):
        x.normal_()
        want = step([p.clone() for p in start])
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(held[turn % 2], want)


@pytest.mark.parametrize("device", EACH)
def test_refusals(device):
    D, N = 64, 3
    table, q, k = build_rope_table(16, D).to(device), torch.zeros(N, 4, D, device=device).bfloat16(), torch.zeros(N, 2, D, device=device).bfloat16()
    pool, plain, rows = kv4_pool(4, 16, 2, D, device), torch.zeros(4, 16, 2, D, device=device).bfloat16(), torch.arange(N, device=device).int()
    good = dict(q=q, k=k, v=k, kpool=pool, vpool=pool, rows=rows, positions=rows, table=table)
    w = torch.ones(D, device=device)
    one = kv4_pool(4, 16, 1, D, device)
    for bad in (dict(q=q[0]), dict(q=q[:2]), dict(k=k[..., :32], v=k[..., :32]), dict(v=k[:, :1]), dict(q=q.half()), dict(k=k.float(), v=k.float()),
                dict(q=q.half(), k=k.half(), v=k.half()), dict(vpool=kv4_pool(5, 16, 2, D, device)), dict(kpool=pool[..., :-1], vpool=pool[..., :-1]),
                dict(kpool=plain[:, :, :1], vpool=plain[:, :, :1]), dict(kpool=one, vpool=one), dict(kpool=plain.float(), vpool=plain.float()),
                dict(kpool=plain), dict(rows=rows.long()), dict(rows=rows[:2]), dict(positions=rows.float()), dict(table=table.half()),
                dict(table=table[:, :32]), dict(q_weight=w), dict(q_weight=w, k_weight=w[:32]), dict(q_weight=w.half(), k_weight=w.half())):
        with pytest.raises(ValueError):
            paged_kv_append(**good | bad)
    for shape in ((4, 8, 2, 64), (4, 24, 2, 64), (4, 16, 2, 96)):
        with pytest.raises(ValueError):
            kv4_pool(*shape)
    for bad in ((pool, pool, rows.long(), D), (pool, pool[:2], rows, D), (pool, pool, rows, 128), (pool, pool, rows, 96), (pool.int(), pool.int(), rows, D)):
        with pytest.raises(ValueError):
            kv4_read(*bad)
    batch = RaggedBatch.build([3], [0], [0], device, [[1]], 16)
    good = dict(q=q, kpool=pool, vpool=pool, batch=batch, scale=0.1, window=0)
    wide = RaggedBatch.build([3], [0], [0], device, [[1]], 32)
    for bad in (dict(q=q[:2]), dict(q=q[:, :3]), dict(q=torch.zeros(N, 4, 96, device=device)), dict(vpool=pool[:3]), dict(window=-1),
                dict(kpool=pool.int(), vpool=pool.int()), dict(kpool=pool[0], vpool=pool[0]), dict(batch=wide),
                dict(batch=RaggedBatch.build([3], [0], [0], device))):
        with pytest.raises(ValueError):
            paged_attention_4bit(**good | bad)
    few = RaggedBatch.build([1, 2], [0, 0], [0, 1], device, [[1], [2]], 16)
    short = RaggedBatch.build([3], [15], [0], device, [[1, 2]], 16)
    few.block_tables, short.block_tables = few.block_tables[:1], short.block_tables[:, :1].contiguous()
    for bad in (few, short):
        with pytest.raises(ValueError):
            paged_attention_4bit(**good | dict(batch=bad))
    if device == "cuda":
        many = torch.zeros(1, device=device).int().expand(1 << 26)   # tokens of a launch's threads
        heads = q[:1, :1].expand(1 << 26, 1, D)
        with pytest.raises(ValueError):
            paged_kv_append(heads, heads, heads, one, one, many, many, table)
        room = torch.zeros(pool.numel() + 8, dtype=torch.uint8, device=device)
        apart = room[8:].view(pool.shape)
        for call in (lambda: paged_attention_4bit(**good | dict(kpool=apart, vpool=apart)), lambda: kv4_read(apart, apart, rows, D),
                     lambda: paged_kv_append(q, k, k, apart, apart, rows, rows, table)):
            with pytest.raises(ValueError):
                call()
        with pytest.raises(ValueError):
            paged_attention_4bit(**good | dict(q=q.float()))
        with pytest.raises(ValueError):
            paged_kv_append(q, k, k, pool, pool, rows, rows, table.cpu())


def test_plan_of_one_long_sequence_beside_many():
    """It is cut, as the others would wait for it; sequences of one length are not."""
    for longest, cut in ((128 * 1024, True), (1024, False)):
        batch = RaggedBatch.build([1] * 200, [longest - 1] + [1023] * 199, list(range(200)), "cpu")
        plan, sizes = batch.row_plan(4, 8)
        steps = [hi - lo for *_, lo, hi, _ in plan[: 6 * sizes[0]].view(-1, 6).tolist()]
        assert (sizes[1] > 0) == cut and max(steps) <= 2 * -(-(199 * 32 + longest // 32) * 8 // 768) and steps == sorted(steps, reverse=True)


@pytest.mark.parametrize("counts,starts", [([1, 1], [4, 0]), ([7, 1, 33, 200, 2], [0, 900, 31, 5, 3000]), ([40], [0]), ([1], [40000])])
@pytest.mark.parametrize("group", [1, 3, 8, 16, 20, 70])
@pytest.mark.parametrize("window", [0, 10, 1000])
def test_plan(counts, starts, group, window):
    """Every key that a new token sees is in exactly one part of the token's one tile; tiles hold their rows; parts are listed with their tiles."""
    batch = RaggedBatch.build(counts, starts, list(range(len(counts))), "cpu")
    for tiles, blocks in (((16, 32, 128), (1024, 512, 512)), ((16, 32, 128), (8, 8, 8)), ((16, 16, 64), (512, 512, 512))):
        plan, sizes = batch.row_plan(group, 2, window, tiles, blocks)
        at, seen = 0, {}
        for kind, rows in enumerate(tiles):
            items, joins, used = sizes[3 * kind: 3 * kind + 3]
            for seq, t0, t1, lo, hi, slot in plan[at: at + 6 * items].view(-1, 6).tolist():
                assert batch.cu_host[seq] <= t0 < t1 <= batch.cu_host[seq + 1] and lo < hi
                assert t1 - t0 == 1 or (t1 - t0) * group <= rows
                seen.setdefault((kind, seq, t0, t1), []).append((lo, hi, slot))
            at += 6 * items
            listed = {(t0, t1): (first, count) for t0, t1, first, count in plan[at: at + 4 * joins].view(-1, 4).tolist()}
            at += 4 * joins
            mine = {k: v for k, v in seen.items() if k[0] == kind}
            assert sum(n for _, n in listed.values()) == used and len(listed) == joins
            taken = sorted(s for v in mine.values() for *_, s in v if s >= 0)
            assert taken == list(range(used))
            for (_, seq, t0, t1), v in mine.items():
                v.sort()
                first = batch.start_host[seq] + t0 - batch.cu_host[seq]
                last = first + t1 - t0 - 1
                assert v[0][0] == (max(0, first - window + 1) // 32 if window else 0) and v[-1][1] == last // 32 + 1
                assert all(a[1] == b[0] for a, b in zip(v, v[1:]))
                if len(v) == 1:
                    assert v[0][2] == -1 and (t0, t1) not in listed
                else:
                    assert len(v) <= 64 and listed[t0, t1] == (v[0][2], len(v)) and [s for *_, s in v] == list(range(v[0][2], v[0][2] + len(v)))
        assert at == plan.numel() and sorted(t for _, _, a, b in seen for t in range(a, b)) == list(range(batch.num_tokens))
