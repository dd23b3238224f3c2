"""Paged keys and values in 4 bits: appending to them, and attention over them (``csrc/serving/cache_append.hip``,
``attention_4bit.hip``).

A number has a sign bit, two exponent bits and a mantissa bit, {0, 0.5, 1, 1.5, 2, 3, 4, 6} and their negatives; 32 neighbouring channels of a
token's head share a power of two, the smallest 2^e with 6 * 2^e at least their largest magnitude, and take the nearest numbers (ties to the
even mantissa): 17/32 byte a channel, 3.8 times the tokens of a bfloat16 cache. A group with a value that is not finite reads as NaN, a value
from 3.5 * 2^126 on as infinite.

``kv4_pool`` makes a pool, uint8 [pages, heads, bytes of a page's head]. Its bytes are tiles of 16 tokens, each tile's codes (two channels a
byte, the lower one in the lower bits), then its scales' bytes e + 127:

* keys: codes [16 tokens, D / 2], scales [16 tokens, D / 32];
* values: codes [4 quads of tokens, 16 lanes, 4 tokens, D / 32 bytes] (a lane has D / 16 neighbouring channels), scales [D / 32, 16 tokens].

Pages are addressed as in every paged cache here (``KVCacheManager``, ``RaggedBatch``): row ``page * page_size + offset``.
"""

from typing import Optional, Tuple

import torch

from ._kernels import serving_kernels, use_serving_hip as use_hip
from .norm_rope import norm_rope_ref
from .ragged import RaggedBatch

__all__ = ["kv4_pool", "kv4_read", "kv4_unpack", "paged_kv_append", "paged_kv_append_ref", "paged_attention_4bit",
           "paged_attention_4bit_ref"]

HEAD_DIMS = (64, 128, 256)
_NUMBERS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# rows of the kernel's tiles by head size, and the blocks that 256 CUs hold at once, by its registers
_TILES = {64: ((16, 32, 128), (1024, 768, 768)), 128: ((16, 32, 128), (768, 512, 512)), 256: ((16, 16, 64), (512, 512, 512))}
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _page_size(pool: torch.Tensor, head_dim: int) -> int:
    """The page size of a pool of 4-bit heads of that size."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"4-bit caches hold heads of 64, 128 or 256 channels, got {head_dim}")
    ps = pool.shape[2] * 32 // (17 * head_dim) if pool.dim() == 3 else 0
    if pool.dtype != torch.uint8 or ps < 16 or ps & (ps - 1) or ps * 17 * head_dim // 32 != pool.shape[2]:
        raise ValueError(f"a 4-bit pool is uint8 [pages, heads, page size * 17 * {head_dim} / 32] with page sizes that are powers of two "
                         f"from 16 on, got {pool.dtype} {tuple(pool.shape)}")
    return ps


def kv4_pool(num_blocks: int, block_size: int, num_heads: int, head_dim: int, device=None) -> torch.Tensor:
    """An empty pool of keys or values: ``num_blocks`` pages of ``block_size`` tokens (a power of two from 16 on), heads of 64, 128 or 256
    channels."""
    if block_size < 16 or block_size & (block_size - 1):
        raise ValueError(f"pages of a 4-bit cache hold a power of two of tokens, 16 at least, got {block_size}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"4-bit caches hold heads of 64, 128 or 256 channels, got {head_dim}")
    return torch.zeros(num_blocks, num_heads, block_size * 17 * head_dim // 32, dtype=torch.uint8, device=device)


def _tiles(pool: torch.Tensor, head_dim: int, values: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """Views of a pool's codes and scale bytes with the tile's token as the last but one (codes of values: four) dimension."""
    P, G, size = pool.shape
    D = head_dim
    t = pool.view(P, G, -1, 17 * D // 2)
    codes, scales = t[..., : 8 * D], t[..., 8 * D:]
    if values:
        return codes.unflatten(-1, (4, 16, 4, D // 32)), scales.unflatten(-1, (D // 32, 16))
    return codes.unflatten(-1, (16, D // 2)), scales.unflatten(-1, (16, D // 32))


def _numbers(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What packed codes [.., D / 2] and scale bytes [.., D / 32] stand for, float32 [.., D]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    grid = torch.tensor(_NUMBERS + tuple(-x for x in _NUMBERS), device=codes.device)
    unit = torch.exp2(scales.float() - 127).masked_fill(scales == 255, float("nan"))
    return (grid[code].unflatten(-1, (-1, 32)) * unit.unsqueeze(-1)).flatten(-2)


def _codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Packed codes and scale bytes of x [.., D], float32 or float64."""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1)
    odd = ~(x.abs() <= torch.finfo(torch.float32).max).all(-1)
    mantissa, e = torch.frexp(most.masked_fill(odd, 0))
    e = (e - 3 + (mantissa > 0.75).int()).masked_fill(mantissa == 0, -126).clamp(min=-126)  # frexp calls 0 a number of 2^0
    a = torch.ldexp(x.abs(), -e.unsqueeze(-1))
    code = sum((a >= b if i % 2 else a > b).byte() for i, b in enumerate(_BORDERS))
    code = code.masked_fill(odd.unsqueeze(-1), 7) | ((x < 0).byte() << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(odd, 255, e + 127).byte()


def kv4_unpack(pool: torch.Tensor, head_dim: int, values: bool) -> torch.Tensor:
    """The numbers of a whole pool, float32 [pages, page size, heads, head_dim]; ``values`` says which of the two layouts it has."""
    _page_size(pool, head_dim)
    codes, scales = _tiles(pool, head_dim, values)
    if values:
        codes, scales = codes.transpose(-3, -2).flatten(-2), scales.transpose(-1, -2)
        codes = codes.flatten(3, 4)
    x = _numbers(codes, scales)  # [pages, heads, tiles, 16, D]
    return x.flatten(2, 3).transpose(1, 2)


def kv4_read(kpool: torch.Tensor, vpool: torch.Tensor, rows: torch.Tensor, head_dim: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The numbers that rows (int32 [N]) of a layer's pools hold: keys and values, bfloat16 [N, heads, head_dim] (which has every one of them
    but products below its smallest). NaN for a row that the pools do not have."""
    if use_hip(kpool):
        return tuple(serving_kernels().kv4_read(kpool, vpool, rows, head_dim))
    ps = _page_size(kpool, head_dim)
    if vpool.shape != kpool.shape or vpool.dtype != torch.uint8:
        raise ValueError(f"both pools have one shape, got {tuple(kpool.shape)} and {tuple(vpool.shape)}")
    if rows.dtype != torch.int32 or rows.dim() != 1:
        raise ValueError(f"rows must be int32 [N], got {rows.dtype} {tuple(rows.shape)}")
    here = (rows >= 0) & (rows < kpool.shape[0] * ps)
    at = torch.where(here, rows, 0).long()
    return tuple(kv4_unpack(p, head_dim, v).flatten(0, 1)[at].masked_fill(~here[:, None, None], float("nan")).bfloat16()
                 for p, v in ((kpool, False), (vpool, True)))


def paged_kv_append_ref(q, k, v, kpool, vpool, rows, positions, table, q_weight=None, k_weight=None, eps=1e-6):
    four = kpool.dtype == torch.uint8
    out = norm_rope_ref(q, q_weight, table, positions, eps).to(q.dtype)
    k = norm_rope_ref(k, k_weight, table, positions, eps, torch.float64 if four else torch.float32)
    ps = _page_size(kpool, q.shape[-1]) if four else kpool.shape[1]
    here = (rows >= 0) & (rows < kpool.shape[0] * ps)
    at = rows[here].long()
    if not four:
        kpool.view(-1, *kpool.shape[2:])[at] = k[here].to(kpool.dtype)
        vpool.view(-1, *vpool.shape[2:])[at] = v[here]
        return out
    page, tile, t = at // ps, at % ps // 16, at % 16
    for pool, x, values in ((kpool, k, False), (vpool, v.float(), True)):
        codes, scales = _codes(x[here])
        to_codes, to_scales = _tiles(pool, q.shape[-1], values)
        if values:
            to_codes[page, :, tile, t // 4, :, t % 4] = codes.unflatten(-1, (16, -1))
            to_scales[page, :, tile, :, t] = scales
        else:
            to_codes[page, :, tile, t] = codes
            to_scales[page, :, tile, t] = scales
    return out


def _check_append(q, k, v, kpool, vpool, rows, positions, table, q_weight, k_weight):
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q [N, H, D] and k, v [N, G, D] expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float32) or not q.dtype == k.dtype == v.dtype:
        raise ValueError(f"q, k and v must be bfloat16 or float32 and of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    N, D = q.shape[0], q.shape[2]
    if kpool.shape != vpool.shape or kpool.dtype != vpool.dtype or not (kpool.is_contiguous() and vpool.is_contiguous()):
        raise ValueError(f"both pools must be contiguous and of one shape and type, got {kpool.dtype} {tuple(kpool.shape)} and "
                         f"{vpool.dtype} {tuple(vpool.shape)}")
    if kpool.dtype == torch.uint8:
        _page_size(kpool, D)
        heads = kpool.shape[1]
    else:
        if kpool.dim() != 4 or kpool.dtype != k.dtype or kpool.shape[3] != D or D % 16 or D > 512:
            raise ValueError(f"pools must be [pages, page size, heads, {D}] of the keys' type, head sizes multiples of 16 up to 512, got "
                             f"{kpool.dtype} {tuple(kpool.shape)}")
        heads = kpool.shape[2]
    if heads != k.shape[1]:
        raise ValueError(f"the pools hold {heads} heads, there are {k.shape[1]}")
    for name, t in (("rows", rows), ("positions", positions)):
        if t.dtype != torch.int32 or t.numel() != N:
            raise ValueError(f"{name} must be int32, one a token, got {t.dtype} {tuple(t.shape)}")
    if table.dim() != 2 or table.shape[1] != D or table.dtype != torch.float32:
        raise ValueError(f"table must be float32 [positions, {D}], got {table.dtype} {tuple(table.shape)}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("both weights or none")
    if q_weight is not None and (q_weight.shape != (D,) or k_weight.shape != (D,) or q_weight.dtype != k_weight.dtype
                                 or q_weight.dtype not in (q.dtype, torch.float32)):
        raise ValueError(f"weights must be [{D}], of the queries' type or float32")


def paged_kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor, rows: torch.Tensor,
                    positions: torch.Tensor, table: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                    k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """New tokens on their way into a paged cache, in one launch: q [N, H, D] and k [N, G, D] are divided by their heads' root mean square and
    multiplied by ``q_weight`` / ``k_weight`` [D] (if both are given) and rotated by ``positions`` (pairs ``(i, i + D / 2)``, ``table`` of
    ``build_rope_table``); keys and values [N, G, D] go to pool rows ``rows``. Returns the queries, contiguous in q's type.

    Types are bfloat16 or float32 (token strides of q, k and v are free), weights of the same type or float32, positions and rows int32 [N].
    Pools are [pages, page size, G, D] of the keys' type (D a multiple of 16 up to 512), or 4-bit ones of ``kv4_pool``. A row that the pools do
    not have, as -1 for a padding token, is not written; no two tokens may have the same one. A position that the table does not have gives
    NaN."""
    if use_hip(q):  # the arguments are looked over there: it takes the host 1 us for 6
        return serving_kernels().paged_kv_append(q, k, v, kpool, vpool, rows, positions, table, q_weight, k_weight, eps)
    _check_append(q, k, v, kpool, vpool, rows, positions, table, q_weight, k_weight)
    return paged_kv_append_ref(q, k, v, kpool, vpool, rows.reshape(-1), positions.reshape(-1), table, q_weight, k_weight, eps)


def paged_attention_4bit_ref(q, kpool, vpool, batch: RaggedBatch, scale: float, window: int = 0):
    N, H, D = q.shape
    k, v = kv4_unpack(kpool, D, False), kv4_unpack(vpool, D, True)
    out = torch.empty(N, H, D, dtype=torch.float32, device=q.device)
    for i in range(batch.num_seqs):
        lo, hi, s0 = batch.cu_host[i], batch.cu_host[i + 1], batch.start_host[i]
        L = s0 + hi - lo
        pages = batch.block_tables[i, : -(-L // batch.page_size)].long()
        here = (pages >= 0) & (pages < k.shape[0])
        kk, vv = (x[pages * here].masked_fill(~here[:, None, None, None], float("nan")).flatten(0, 1)[:L].repeat_interleave(H // x.shape[2], 1)
                  .transpose(0, 1) for x in (k, v))
        at, key = torch.arange(s0, L, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
        seen = key <= at
        if window > 0:
            seen = seen & (at - key < window)
        p = torch.softmax((q[lo:hi].float().transpose(0, 1) @ kk.transpose(1, 2) * scale).masked_fill(~seen, float("-inf")), -1)
        shown = (seen.float() @ (~vv.isfinite()).float()) > 0  # a weight of 0 hides what is not seen
        out[lo:hi] = (p @ vv.nan_to_num(0.0, 0.0, 0.0)).masked_fill(shown, float("nan")).transpose(0, 1)
    return out.to(q.dtype)


def paged_attention_4bit(q: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor, batch: RaggedBatch, scale: float,
                         window: int = 0) -> torch.Tensor:
    """``paged_attention`` over a 4-bit cache, which already holds the step's keys (``paged_kv_append`` runs first): q [N, H, D] in bfloat16
    (token stride free), causal, limited to a sliding ``window`` if it is not 0; query head ``h`` reads head ``h // (H / G)``. Single tokens and
    prompt portions of any lengths in one call. Returns [N, H, D] in q's type. Scores, sums and the accumulation are float32; a weight is
    two bfloat16 pieces for its product, 16 bits, whatever shares the step. A page number that the pools do not have gives NaN to the tokens that see
    it. The plan of a step's work is made by the first call with a batch and kept by it, not while a graph is captured."""
    if q.dim() != 3 or q.shape[0] != batch.num_tokens:
        raise ValueError(f"q must be [{batch.num_tokens}, H, D], got {tuple(q.shape)}")
    _, H, D = q.shape
    G = kpool.shape[1] if kpool.dim() == 3 else 0
    if D not in HEAD_DIMS or G == 0 or H % G:
        raise ValueError(f"heads of 64, 128 or 256 channels, the pools' heads shared by as many query heads each, got {H} heads of {D} and pools "
                         f"{tuple(kpool.shape)}")
    if batch.block_tables is None or window < 0:
        raise ValueError("a batch with page tables, and a window of 0 or more")
    if use_hip(q):
        plan, sizes = batch.row_plan(H // G, G, window, *_TILES[D])
        return serving_kernels().paged_attention_4bit(q, kpool, vpool, batch.block_tables, batch.positions, plan, sizes, scale, window, batch.page_size)
    ps = _page_size(kpool, D)
    tables = batch.block_tables.shape
    if (vpool.shape != kpool.shape or vpool.dtype != torch.uint8 or batch.page_size != ps or tables[0] < batch.num_seqs
            or tables[1] * ps < batch.max_total):
        raise ValueError(f"a table row of all its pages a sequence, and both pools have one shape and the batch's pages of {batch.page_size} tokens, got {tuple(kpool.shape)} and {tuple(vpool.shape)}")
    return paged_attention_4bit_ref(q, kpool, vpool, batch, scale, window)
