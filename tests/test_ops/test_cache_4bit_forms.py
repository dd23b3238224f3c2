"""Attention over 4-bit caches in each form that its kernels have: by the rows that a sequence's new tokens make, and by what shares their step.

A form is a step's new tokens and cached tokens, with the kind of tile that the step's plan is to give it (0: the fewest rows, 1, 2: the most)."""

import math

import pytest
import torch

from colossalai_amd.ops import kv4_pool, paged_attention_4bit
from colossalai_amd.ops.cache_4bit import _TILES, _tiles, kv4_unpack
from colossalai_amd.ops.ragged import RaggedBatch

gpu = pytest.mark.gpu
GROUP, HEADS, PAGE = 4, 2, 16
FORMS = {"single": ([1, 1, 1], [700, 33, 2000], {0}), "single beside a short portion": ([1, 10, 1], [700, 300, 40], {1}),
         "short portion": ([10], [500], {1}), "portions": ([70, 150], [300, 90], {2}), "all": ([1, 150, 10], [700, 90, 300], {1, 2})}
forms = pytest.mark.parametrize("form", FORMS)
sizes = pytest.mark.parametrize("D", [64, 128, 256])


def _step(form, D, device="cuda", seed=0):
    """The step's batch, the pages of its sequences, queries, and pools of random numbers of about one size."""
    counts, starts, kinds = FORMS[form]
    g = torch.Generator().manual_seed(seed)
    need = [-(-(a + b) // PAGE) for a, b in zip(counts, starts)]
    order, tables = torch.randperm(sum(need) + 2, generator=g).tolist(), []
    for n in need:
        tables.append([order.pop() for _ in range(n)])
    batch = RaggedBatch.build(counts, starts, list(range(len(counts))), device, tables, PAGE)
    items = batch.row_plan(GROUP, HEADS, 0, *_TILES[D])[1][:9:3]
    assert {k for k in range(3) if items[k]} == kinds
    pools = []
    for values in (False, True):
        pool = torch.randint(0, 256, kv4_pool(sum(need) + 2, PAGE, HEADS, D).shape, generator=g).byte()
        scales = _tiles(pool, D, values)[1]
        scales.copy_(torch.randint(124, 129, scales.shape, generator=g).byte())
        pools.append(pool.to(device))
    q = torch.randn(sum(counts), GROUP * HEADS, D, generator=g).to(device, torch.bfloat16)
    return batch, tables, q, pools


def _exact(batch, tables, q, pools, scale):
    """Of each sequence: outputs in 64 bits, sums of p |v|, and the largest scale * sum |q k|; all [heads, tokens, D] but the last."""
    D = q.shape[-1]
    k, v = (kv4_unpack(p, D, x).double() for p, x in zip(pools, (False, True)))
    for i, t in enumerate(tables):
        lo, hi, s = batch.cu_host[i], batch.cu_host[i + 1], batch.start_host[i]
        kk, vv = (x[torch.tensor(t, device=q.device)].flatten(0, 1)[: s + hi - lo].repeat_interleave(GROUP, 1).transpose(0, 1) for x in (k, v))
        qq = q[lo:hi].double().transpose(0, 1)
        row, key = torch.arange(s, s + hi - lo, device=q.device)[:, None], torch.arange(s + hi - lo, device=q.device)[None]
        p = torch.softmax((qq @ kk.transpose(1, 2) * scale).masked_fill(key > row, -math.inf), -1)
        yield slice(lo, hi), p @ vv, p @ vv.abs(), float(((qq.abs() @ kk.abs().transpose(1, 2)) * scale).amax())


@gpu
@forms
@sizes
def test_weights_have_16_bits(form, D):
    """The output is rounded once, 2^-8 of it. A weight is two bfloat16 pieces: the first leaves at most 2^-8 of it, the second 2^-8 of that. A
    score's float32 error, D + 2 roundings of scale * sum |q k|, moves a weight by as much of itself, its exponential has 2^-22, and the sums over L
    keys have at most L 2^-24 each. Where an output is a small difference of its terms, as some of these are, 2^-8 of the terms does not pass."""
    batch, tables, q, pools = _step(form, D)
    scale = D ** -0.5
    got = paged_attention_4bit(q, *pools, batch, scale).double()
    for rows, want, near, size in _exact(batch, tables, q, pools, scale):
        keys = max(s + b - a for s, a, b in zip(batch.start_host, batch.cu_host, batch.cu_host[1:]))
        slack = 2.0 ** -16 + 2.0 ** -22 + 2 * (D + 2) * 2.0 ** -24 * size + 2 * keys * 2.0 ** -24
        off = (got[rows].transpose(0, 1) - want).abs() - 2.0 ** -8 * want.abs() - slack * near
        assert (off <= 0).all(), f"{float((off / near).max()):.2e} of the terms over the bound"
