"""Attention over 4-bit caches in each form that its kernels have: by the rows that a sequence's new tokens make, and by what shares their step.

A form is a step's new tokens and cached tokens, with the kind of tile that the step's plan is to give it (0: the fewest rows, 1, 2: the most)."""

import math

import pytest
import torch

from colossalai_amd.ops import kv4_pool, paged_attention_4bit, paged_kv_append
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


@gpu
@forms
@sizes
def test_a_token_is_its_own_affair(form, D):
    """Whatever the others of its step ask for, to the last bit: their scores, up to hundreds, come at other keys."""
    batch, tables, q, pools = _step(form, D)
    want = paged_attention_4bit(q, *pools, batch, D ** -0.5)
    for every in (2, 3):
        others = torch.arange(len(q), device="cuda") % every != 0
        again = q.clone()
        again[others] = 40 * again[others].flip(0)
        got = paged_attention_4bit(again, *pools, batch, D ** -0.5)
        assert torch.equal(got[~others], want[~others])
        again = q.clone()
        again[:, 1::2] *= 40  # heads beside it
        assert torch.equal(paged_attention_4bit(again, *pools, batch, D ** -0.5)[:, ::2], want[:, ::2])


def _put(pools, tables, values, seq, key, head, code, byte, group=1):
    """One channel's code, all others of its group 0, and the group's scale byte, for a key of a sequence."""
    pool = pools[values]
    D = pool.shape[2] * 32 // (17 * PAGE)
    codes, scales = _tiles(pool, D, values)
    page, t = tables[seq][key // PAGE], key % PAGE
    mine = codes[page, head, 0, t // 4, :, t % 4] if values else codes[page, head, 0, t]  # [16, D / 32] or [D / 2]
    flat = mine.reshape(-1).clone()
    flat[group * 16: group * 16 + 16] = 0
    flat[group * 16 + 5] = code
    mine.copy_(flat.view(mine.shape))
    (scales[page, head, 0, :, t] if values else scales[page, head, 0, t])[group] = byte


NOT_FINITE = [(7, 255), (0, 255), (6, 253), (15, 253), (4, 254), (13, 254)]
FINITE = [(5, 253), (13, 253), (3, 254), (11, 254), (7, 252)]


@sizes
@pytest.mark.parametrize("code,byte", NOT_FINITE)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_values_that_are_not_finite_stay_with_the_tokens_that_see_them(code, byte, device, D):
    """NaN by the scale, infinite by the number. Tokens ahead of it, and those whose window it has left, are what they were; those that
    see it are not finite in its channel. In steps that all tokens see, and in those that some do not."""
    for form in FORMS:
        batch, tables, q, clean = _step(form, D, device)
        for window in (0, 20):
            want = paged_attention_4bit(q, *clean, batch, D ** -0.5, window)
            assert want.isfinite().all()
            for seq in range(batch.num_seqs):
                lo, hi, start = batch.cu_host[seq], batch.cu_host[seq + 1], batch.start_host[seq]
                at = torch.arange(start, start + hi - lo, device=device)
                for key in {0, start // 2, max(0, start - 19), start, start + (hi - lo) // 2, start + hi - lo - 1}:
                    pools = [p.clone() for p in clean]
                    _put(pools, tables, True, seq, key, 1, code, byte)
                    got = paged_attention_4bit(q, *pools, batch, D ** -0.5, window)
                    sees = torch.zeros(len(q), dtype=torch.bool, device=device)
                    sees[lo:hi] = (key <= at) & ((at - key < window) | (window == 0))
                    assert torch.equal(got[~sees], want[~sees]) and torch.equal(got[sees, :GROUP], want[sees, :GROUP]), (form, window, seq, key)
                    assert not got[sees, GROUP:, 32 + 10].isfinite().any(), (form, window, seq, key)


@sizes
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_keys_that_are_not_finite_show_whatever_the_queries_sign(sign, device, D):
    """A group with one infinity is code 7 there and 0 elsewhere, at scale byte 255: no key that scores of minus infinity would hide."""
    for form in FORMS:
        batch, tables, q, clean = _step(form, D, device)
        q = sign * q.abs()
        want = paged_attention_4bit(q, *clean, batch, D ** -0.5)
        for seq in range(batch.num_seqs):
            lo, hi, start = batch.cu_host[seq], batch.cu_host[seq + 1], batch.start_host[seq]
            for key in {0, start // 2, start, start + hi - lo - 1}:
                for code in (7, 0):
                    pools = [p.clone() for p in clean]
                    _put(pools, tables, False, seq, key, 1, code, 255)
                    got = paged_attention_4bit(q, *pools, batch, D ** -0.5)
                    sees = torch.zeros(len(q), dtype=torch.bool, device=device)
                    sees[lo:hi] = torch.arange(start, start + hi - lo, device=device) >= key
                    assert torch.equal(got[~sees], want[~sees]) and torch.equal(got[sees, :GROUP], want[sees, :GROUP]), (form, seq, key)
                    assert got[sees, GROUP:].isnan().all(), (form, seq, key)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@sizes
def test_an_appended_infinity_shows(device, D):
    """From the append to the attention: one infinite channel of a key, queries of one sign against it."""
    batch = RaggedBatch.build([1], [40], [0], device, [[2, 0, 1]], PAGE)
    pools = [kv4_pool(3, PAGE, HEADS, D, device) for _ in range(2)]
    table = torch.cat([torch.ones(64, D // 2), torch.zeros(64, D // 2)], 1).to(device)  # turned by nothing
    x = torch.ones(41, GROUP * HEADS + 2 * HEADS, D, device=device).bfloat16()
    q, k, v = x.split([GROUP * HEADS, HEADS, HEADS], 1)
    k[7, 1, 3] = math.inf
    at = torch.arange(41, device=device).int()
    rows = torch.tensor([2, 0, 1], device=device).int()[at // PAGE] * PAGE + at % PAGE
    for sign in (-1, 1):
        last = paged_kv_append(sign * q.contiguous(), k, v, *pools, rows, at, table)[-1:]
        got = paged_attention_4bit(last, *pools, batch, D ** -0.5)
        assert (got[:, :GROUP] == 1).all() and got[:, GROUP:].isnan().all()


@sizes
@pytest.mark.parametrize("page", [-1, -5, 10 ** 6])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_pages_that_the_pool_does_not_have(page, device, D):
    """NaN to the tokens that see a key of one, and nothing to others, in every form: no page counted from the end."""
    for form in FORMS:
        batch, tables, q, pools = _step(form, D, device)
        for window in (0, 20):
            want = paged_attention_4bit(q, *pools, batch, D ** -0.5, window)
            for seq in range(batch.num_seqs):
                lo, hi, start = batch.cu_host[seq], batch.cu_host[seq + 1], batch.start_host[seq]
                at = torch.arange(start, start + hi - lo, device=device)
                for i in {0, start // PAGE, len(tables[seq]) - 1, max(0, start - 20) // PAGE}:
                    held = batch.block_tables[seq, i].item()
                    batch.block_tables[seq, i] = page
                    got = paged_attention_4bit(q, *pools, batch, D ** -0.5, window)
                    batch.block_tables[seq, i] = held
                    sees = torch.zeros(len(q), dtype=torch.bool, device=device)
                    sees[lo:hi] = (at >= i * PAGE) & ((at - (i + 1) * PAGE + 1 < window) | (window == 0))
                    assert torch.equal(got[~sees], want[~sees]) and got[sees].isnan().all(), (form, window, seq, i)


@sizes
@pytest.mark.parametrize("code,byte", FINITE)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_the_largest_values_that_are_finite(code, byte, device, D):
    """They are no more than values: of other tokens nothing changes, and of those that see one its channel alone."""
    batch, tables, q, clean = _step("all", D, device)
    want = paged_attention_4bit(q, *clean, batch, D ** -0.5)
    for seq, key in ((0, 700), (1, 0), (1, 90), (1, 131), (1, 239), (2, 304)):
        pools, zeros = [p.clone() for p in clean], [p.clone() for p in clean]
        _put(pools, tables, True, seq, key, 1, code, byte)
        _put(zeros, tables, True, seq, key, 1, 0, 127)
        got, without = (paged_attention_4bit(q, *p, batch, D ** -0.5) for p in (pools, zeros))
        other = torch.ones(D, dtype=torch.bool, device=device)
        other[32 + 10] = False
        assert torch.equal(got[..., other], without[..., other])
        sees = torch.zeros(len(q), dtype=torch.bool, device=device)
        lo, hi = batch.cu_host[seq], batch.cu_host[seq + 1]
        sees[lo:hi] = torch.arange(hi - lo, device=device) + batch.start_host[seq] >= key
        assert torch.equal(got[~sees], want[~sees]) and not got[sees, GROUP:, 32 + 10].isnan().any()


def test_plans_of_other_steps_are_others():
    """A batch keeps a plan by all that it was asked for: steps of 16 keys are twice as many, and longer parts are fewer."""
    batch = RaggedBatch.build([1, 1], [999, 4000], [0, 1], "cpu")
    ends = lambda plan, sizes: plan[: 6 * sizes[0]].view(-1, 6)[:, 4].max().item()  # noqa: E731
    first = batch.row_plan(4, 2)
    assert ends(*first) == -(-4001 // 32) and ends(*batch.row_plan(4, 2, step=16)) == -(-4001 // 16)
    assert batch.row_plan(4, 2, least=1000)[1][0] == 2 < first[1][0]
    assert batch.row_plan(4, 2) is first


@sizes
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_scale_bytes_of_zeros(device, D):
    """The smallest power of two that clips nothing of a group of zeros is the smallest there is, byte 1; so it is for numbers up to 6 * 2^-126."""
    pools = [kv4_pool(1, PAGE, HEADS, D, device).fill_(99) for _ in range(2)]
    x = torch.zeros(PAGE, HEADS, D, device=device)
    x[1], x[2], x[3] = 2.0 ** -126, 6 * 2.0 ** -126, 6.5 * 2.0 ** -126
    at = torch.arange(PAGE, device=device).int()
    table = torch.cat([torch.ones(PAGE, D // 2), torch.zeros(PAGE, D // 2)], 1).to(device)
    paged_kv_append(torch.zeros(PAGE, 4, D, device=device), x, x, *pools, at, at, table)
    for values in (False, True):
        codes, scales = _tiles(pools[values], D, values)
        by_token = (scales.transpose(-1, -2) if values else scales)[0, :, 0]
        assert (by_token[:, 3] == 2).all() and (by_token[:, :3] == 1).all() and (by_token[:, 4:] == 1).all()
        token = (lambda t: codes[0, :, 0, t // 4, :, t % 4]) if values else (lambda t: codes[0, :, 0, t])
        assert (token(0) == 0).all() and (token(1) == 0x22).all() and (token(2) == 0x77).all()
