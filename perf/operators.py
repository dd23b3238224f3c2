"""The operators of serving and training models whose queries and keys are normed head by head, and of caches held in 4 bits.

Three operators that hang together, each with a plain form in elementary torch operations:

* ``qkv_norm_rope``: a packed projection ``[q | k | v]`` is split, each query and key head is divided by its root mean
  square, multiplied by a learned weight and rotated by its position, in one pass, with the backward pass ("train");
* ``paged_kv_append``: the same on the way into a paged cache: queries come back, keys and values go to their pages, in
  the activations' type or in 4 bits ("append");
* ``paged_attention_4bit``: attention of single tokens and prompt portions over such a 4-bit cache ("attend").

"step" is the append and the attention of one engine step, as they are used together.

A 4-bit cache holds numbers of one sign bit, two exponent bits and one mantissa bit, {0, 0.5, 1, 1.5, 2, 3, 4, 6}, and a
power of two for each 32 channels of a token's head: the smallest 2^e with 6 * 2^e >= the largest magnitude, nearest
numbers, ties to the even mantissa. The scale's byte is e + 127, at least 1. A pool is [pages, heads, bytes]; a page's head is
tiles of 16 tokens, a tile's codes (two channels a byte, the lower one in the lower bits) and then its scale bytes:

* keys: codes [16 tokens, D / 2], scales [16 tokens, D / 32];
* values: codes [4 quads of tokens, 16 lanes, 4 tokens, D / 32 bytes] (a lane has D / 16 neighbouring channels), scales
  [D / 32 groups, 16 tokens].
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a small model's step: latency counts
        dict(name="train_small", kind="train", batch=2, seq=256, heads=8, kv_heads=2, dim=64, dtype="bf16", packed=False),
        # the 8B decoder with normed heads at its full context
        dict(name="train_8b", kind="train", batch=4, seq=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", packed=False),
        # packed samples (positions start again at each), odd sizes, 32-bit training
        dict(name="train_packed_fp32", kind="train", batch=1, seq=5003, heads=12, kv_heads=4, dim=96, dtype="fp32", packed=True),
        # the decode step of 48 sequences into a 4-bit cache
        dict(name="append_decode", kind="append", tokens=48, heads=32, kv_heads=8, dim=128, page=16, bits=4, norm=True, prompt=False),
        # prompts into a 4-bit cache
        dict(name="append_prompt", kind="append", tokens=8192, heads=32, kv_heads=8, dim=128, page=64, bits=4, norm=True, prompt=True),
        # prompts of a model without norms into a 16-bit cache (the 7B decoder with 28 query heads)
        dict(name="append_16bit", kind="append", tokens=4099, heads=28, kv_heads=4, dim=128, page=16, bits=16, norm=False, prompt=True),
        # one short conversation: the smallest call
        dict(name="attend_one", kind="attend", seqs=1, new=1, cached=200, heads=16, kv_heads=2, dim=64, page=16, window=0),
        # decode over long contexts: the cache's bytes
        dict(name="attend_long", kind="attend", seqs=16, new=1, cached=32768, heads=32, kv_heads=8, dim=128, page=64, window=0),
        # decode of many sequences of all lengths, a sliding window
        dict(name="attend_window", kind="attend", seqs=61, new=1, cached=9000, heads=28, kv_heads=4, dim=128, page=16, window=4096),
        # portions of prompts over what the cache holds already
        dict(name="attend_portions", kind="attend", seqs=4, new=1000, cached=4000, heads=32, kv_heads=8, dim=128, page=32, window=0),
        # the whole of an engine's step: append, then attend
        dict(name="step_decode", kind="step", seqs=32, new=1, cached=8192, heads=32, kv_heads=8, dim=128, page=16, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "append", "attend", "attend", "step"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8] if kv < 8 else [1, 2, 4])
    if kind == "train":
        dim, dtype = rng.choice([64, 96, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 3 * 10 ** 8 // ((heads + 2 * kv) * dim * (4 if dtype == "fp32" else 2))  # tokens
        seq = _log_int(rng, 17, min(8192, most))
        packed = rng.random() < 0.3
        return dict(kind=kind, batch=1 if packed else max(1, min(_log_int(rng, 64, 16384), most) // seq), seq=seq, heads=heads,
                    kv_heads=kv, dim=dim, dtype=dtype, packed=packed)
    dim, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64])
    if kind == "append":
        prompt = rng.random() < 0.6
        return dict(kind=kind, tokens=_log_int(rng, 16, 8192) if prompt else _log_int(rng, 1, 200), heads=heads, kv_heads=kv,
                    dim=dim, page=page, bits=rng.choice([4, 4, 16]), norm=rng.random() < 0.7, prompt=prompt)
    window = rng.choice([0, 0, 0, 128, 1000, 4096])
    if kind == "attend" and rng.random() < 0.4:
        most = min(2048, 2 ** 23 // (heads * dim))  # new tokens
        new = _log_int(rng, 2, most // 2)
        return dict(kind=kind, seqs=max(1, min(8, most // new)), new=new, cached=_log_int(rng, 1, 4096), heads=heads,
                    kv_heads=kv, dim=dim, page=page, window=window)
    cached = _log_int(rng, 16, 32768)
    return dict(kind=kind, seqs=rng.randint(1, max(1, min(64, 2 ** 21 // (cached * kv)))), new=1, cached=cached, heads=heads,
                kv_heads=kv, dim=dim, page=page, window=window)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(1000003 * seed + 29)


def _table(rows, dim):
    """Cosines and sines of the first `rows` positions, [rows, dim] = [cos | sin], as models keep them."""
    freq = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def _weight(g, dim, dtype):
    return (1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype)


def _projection(g, rows, heads, kv, dim, dtype):
    """A projection's output: keys have a few channels that are larger than the others, as trained models' keys do."""
    x = torch.randn(rows, heads + 2 * kv, dim, generator=g, device="cuda")
    gain = torch.exp(0.5 * torch.randn(kv, dim, generator=g, device="cuda"))
    x[:, heads: heads + kv] *= gain
    return x.reshape(rows, -1).to(dtype)


def _samples(total, seed):
    """Lengths of up to 32 samples, `total` tokens together."""
    g, left, out = _gen(seed, "cpu"), total, []
    while left > 0:
        out.append(min(left, 1 + int(total * float(torch.rand((), generator=g)) ** 3)) if len(out) < 31 else left)
        left -= out[-1]
    return out


def _batch(case, seed):
    """New and cached tokens of each sequence, page tables in the order that a used pool gives, and the pages there are."""
    g = _gen(seed, "cpu")
    u = torch.rand(case["seqs"], generator=g).tolist()
    starts = [max(0, int(case["cached"] * (0.25 + 0.75 * x))) for x in u]
    starts[0] = case["cached"]
    counts = [max(1, int(case["new"] * (1.0 - 0.07 * (3 * i % 8)))) for i in range(case["seqs"])]
    need = [-(-(s + n) // case["page"]) for s, n in zip(starts, counts)]
    order = torch.randperm(sum(need) + 3, generator=g).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at: at + n])
        at += n
    return counts, starts, tables, len(order)


def _cache(g, case, pages):
    """The numbers in a cache, as codes [pages, page, heads, dim] and scale bytes [pages, page, heads, dim / 32]."""
    out = []
    for gain in (0.7, 0.0):
        x = torch.randn(pages, case["page"], case["kv_heads"], case["dim"], generator=g, device="cuda")
        x *= torch.exp(gain * torch.randn(case["kv_heads"], case["dim"], generator=g, device="cuda"))
        x = x.view(*x.shape[:3], -1, 32)
        m, e = torch.frexp(x.abs().amax(-1))
        e = e - 3 + (m > 0.75).int()
        a = torch.ldexp(x.abs(), -e[..., None])
        code = torch.bucketize(a, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")).byte()
        code |= (x < 0).byte() << 3
        out += [code.flatten(-2), (e + 127).byte()]
        del x, a
    return out


def _lay_keys(codes, scales):
    p, ps, h, d = codes.shape
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).view(p, ps // 16, 16, h, d // 2).permute(0, 3, 1, 2, 4)
    s = scales.view(p, ps // 16, 16, h, d // 32).permute(0, 3, 1, 2, 4)
    return torch.cat([packed.reshape(p, h, ps // 16, -1), s.reshape(p, h, ps // 16, -1)], -1).reshape(p, h, -1)


def _lay_values(codes, scales):
    p, ps, h, d = codes.shape
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).view(p, ps // 16, 4, 4, h, 16, d // 32).permute(0, 4, 1, 2, 5, 3, 6)
    s = scales.view(p, ps // 16, 16, h, d // 32).permute(0, 3, 1, 4, 2)
    return torch.cat([packed.reshape(p, h, ps // 16, -1), s.reshape(p, h, ps // 16, -1)], -1).reshape(p, h, -1)


def prepare(case, seed):
    g = _gen(seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case)
    if case["kind"] == "train":
        dtype, rows = TYPES[case["dtype"]], case["batch"] * case["seq"]
        s["qkv"] = _projection(g, rows, h, kv, d, dtype).view(case["batch"], case["seq"], -1).requires_grad_()
        s["weights"] = [_weight(g, d, dtype).requires_grad_() for _ in range(2)]
        s["grads"] = [torch.randn(case["batch"], case["seq"], n, d, generator=g, device="cuda").to(dtype) for n in (h, kv, kv)]
        s["positions"] = None
        if case["packed"]:
            s["positions"] = torch.cat([torch.arange(n, device="cuda") for n in _samples(rows, seed)]).int()
        s["table"] = _table(case["seq"] if not case["packed"] else rows, d)
        return s
    if case["kind"] == "append":
        n, ps = case["tokens"], case["page"]
        if case["prompt"]:  # whole prompts, pages in any order
            lens = _samples(n, seed)
            pos = torch.cat([torch.arange(x) for x in lens])
        else:  # a token of each sequence, somewhere in a page of its own
            lens = [1] * n
            pos = torch.randint(0, 8192, (n,), generator=_gen(seed, "cpu"))
        pages = n // ps + 33 if case["prompt"] else n + 5
        order, rows, at = torch.randperm(pages, generator=_gen(seed, "cpu")), [], 0
        for x in lens:
            i = torch.arange(x) if case["prompt"] else pos[len(rows)] % ps + torch.arange(1)
            rows.append(order[at + i // ps] * ps + i % ps)
            at += -(-x // ps)
        s["rows"], s["positions"] = torch.cat(rows).int().cuda(), pos.int().cuda()
        s["table"] = _table(8192, d)
        s["qkv"] = _projection(g, n, h, kv, d, torch.bfloat16)
        if case["bits"] == 4:
            s["kpool"], s["vpool"] = (torch.ones(pages, kv, ps * 17 * d // 32, dtype=torch.uint8, device="cuda") for _ in range(2))
        else:
            s["kpool"], s["vpool"] = (torch.zeros(pages, ps, kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    else:
        counts, starts, tables, pages = _batch(case, seed)
        codes = _cache(g, case, pages)
        s["kpool"], s["vpool"] = _lay_keys(*codes[:2]), _lay_values(*codes[2:])
        n = sum(counts)
        width = max(len(t) for t in tables)
        s["counts"], s["starts"] = (torch.tensor(x, device="cuda") for x in (counts, starts))
        s["tables"] = torch.tensor([t + [0] * (width - len(t)) for t in tables], device="cuda")
        s["most"], s["length"] = max(counts), max(a + b for a, b in zip(counts, starts))
        s["even"] = min(counts) == max(counts)
        if own:  # an engine has it before the layers run
            from colossalai_amd.ops.ragged import RaggedBatch

            s["batch"] = RaggedBatch.build(counts, starts, list(range(len(counts))), "cuda", tables, case["page"])
        if case["kind"] == "attend":
            s["q"] = (1.5 * torch.randn(n, h, d, generator=g, device="cuda")).to(torch.bfloat16)
            return s
        s["qkv"] = _projection(g, n, h, kv, d, torch.bfloat16)
        s["table"] = _table(s["length"], d)
        s["rows"] = torch.tensor([t[p // case["page"]] * case["page"] + p % case["page"] for c, b, t in zip(counts, starts, tables)
                                  for p in range(b, b + c)], dtype=torch.int32, device="cuda")
        s["positions"] = torch.tensor([p for c, b in zip(counts, starts) for p in range(b, b + c)], dtype=torch.int32, device="cuda")
    if case.get("norm", True):
        s["weights"] = [_weight(g, d, torch.bfloat16) for _ in range(2)]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _normed(x, weight, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.to(x.dtype)


def _rotated(x, table, positions):
    """x [.., tokens, heads, D] in 32 or 64 bits."""
    cos, sin = table[positions.long()].to(x.dtype).chunk(2, -1)
    lo, hi = x.chunk(2, -1)
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _train_plain(s):
    case, qkv = s["case"], s["qkv"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = qkv.float().view(*qkv.shape[:2], -1, d).split([h, kv, kv], 2)
    pos = torch.arange(case["seq"], device="cuda") if s["positions"] is None else s["positions"]
    out = [_rotated(_normed(x, w.float()), s["table"], pos).to(qkv.dtype) for x, w in zip((q, k), s["weights"])]
    out.append(v.to(qkv.dtype))
    return out + list(torch.autograd.grad(out, [qkv, *s["weights"]], s["grads"]))


def _nearest(x):
    """Codes and scale exponents of x [.., D] in 32 or 64 bits."""
    x = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 3 + (m > 0.75).int()).clamp(min=-126)
    a = torch.ldexp(x.abs(), -e[..., None])
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code | (x < 0).byte() << 3).flatten(-2), e


def _number(code, e):
    """What codes [.., D] and exponents [.., D / 32] stand for, in 32 bits."""
    grid = torch.tensor(GRID + tuple(-x for x in GRID), device=code.device)
    return (grid[code.long()].unflatten(-1, (-1, 32)) * torch.exp2(e.float())[..., None]).flatten(-2)


def _append_plain(s):
    """The queries, and keys and values as they are written: codes with exponents, or numbers in the pools' type."""
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = s["qkv"].view(-1, h + 2 * kv, d).split([h, kv, kv], 1)
    four = s["kpool"].dtype == torch.uint8
    q, k = q.float(), k.double() if four else k.float()  # a code is that of the exact key: 32 bits lose what is next to a border
    if "weights" in s:
        q, k = _normed(q, s["weights"][0]), _normed(k, s["weights"][1])
    q, k = (_rotated(x, s["table"], s["positions"]) for x in (q, k))
    return q.to(s["qkv"].dtype), (_nearest(k) if four else k), (_nearest(v.float()) if four else v)


def _write_plain(pool, rows, code, e, values):
    p, kv, size = pool.shape
    d = code.shape[-1]
    ps = size * 32 // (17 * d)
    page, off = rows.long() // ps, rows.long() % ps
    tiles = pool.view(p, kv, ps // 16, -1)
    packed, scale, t = code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).byte(), off % 16
    if values:
        tiles[..., : 8 * d].view(p, kv, ps // 16, 4, 16, 4, d // 32)[page, :, off // 16, t // 4, :, t % 4] = packed.view(-1, kv, 16, d // 32)
        tiles[..., 8 * d:].view(p, kv, ps // 16, d // 32, 16)[page, :, off // 16, :, t] = scale
    else:
        tiles[..., : 8 * d].view(p, kv, ps // 16, 16, d // 2)[page, :, off // 16, t] = packed
        tiles[..., 8 * d:].view(p, kv, ps // 16, 16, d // 32)[page, :, off // 16, t] = scale


def _cached_plain(pool, tables, d, values):
    """The numbers of each sequence's pages, [sequences, heads, tokens, D] in 32 bits."""
    ps = pool.shape[2] * 32 // (17 * d)
    got = pool[tables]  # [B, pages, heads, bytes]
    b, w, kv, _ = got.shape
    got = got.view(b, w, kv, ps // 16, -1).permute(0, 2, 1, 3, 4).reshape(b, kv, w * ps // 16, -1)
    codes, scales = got[..., : 8 * d], got[..., 8 * d:]
    if values:
        codes = codes.reshape(b, kv, -1, 4, 16, 4, d // 32).transpose(4, 5)
        scales = scales.reshape(b, kv, -1, d // 32, 16).transpose(3, 4)
    codes, scales = codes.reshape(b, kv, -1, d // 2), scales.reshape(b, kv, -1, d // 32)
    return _number(torch.stack([codes & 15, codes >> 4], -1).flatten(-2), scales.int() - 127)


def _attend_plain(s, q):
    case = s["case"]
    kv, d = case["kv_heads"], case["dim"]
    b, t = len(s["counts"]), s["most"]
    k, v = _cached_plain(s["kpool"], s["tables"], d, False), _cached_plain(s["vpool"], s["tables"], d, True)
    which = torch.arange(t, device="cuda")[None, :] < s["counts"][:, None]
    padded = torch.zeros(b, t, *q.shape[1:], device="cuda")
    if s["even"]:
        padded = q.float().view(b, t, *q.shape[1:])
    else:
        padded[which] = q.float()
    padded = padded.view(b, t, kv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)  # [B, kv, heads of it x tokens, D]
    scores = (padded @ k.transpose(-1, -2)) * d ** -0.5
    at = (s["starts"][:, None] + torch.arange(t, device="cuda"))[:, None, None, :, None]
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= at
    if case["window"]:
        seen &= key > at - case["window"]
    scores = scores.view(b, kv, -1, t, k.shape[2]).masked_fill_(~seen, -math.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    scores /= scores.sum(-1, keepdim=True)
    out = (scores.view(b, kv, -1, k.shape[2]) @ v).view(b, kv, -1, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, -1, d)
    return (out.reshape(-1, *q.shape[1:]) if s["even"] else out[which]).to(q.dtype)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "train":
        return _train_plain(s)
    if kind == "attend":
        return _attend_plain(s, s["q"])
    q, k, v = _append_plain(s)
    if s["kpool"].dtype != torch.uint8:
        rows = s["rows"].long()
        for pool, x in ((s["kpool"], k), (s["vpool"], v)):
            pool.view(-1, *pool.shape[2:])[rows] = x.to(pool.dtype)
        return q, s["kpool"], s["vpool"]
    _write_plain(s["kpool"], s["rows"], *k, False)
    _write_plain(s["vpool"], s["rows"], *v, True)
    if kind == "step":
        return _attend_plain(s, q)
    return q, _number(*k).to(q.dtype), _number(*v).to(q.dtype)


# ------------------------------------------------------------------------------------------------ the framework's operators
def _run_own(s):
    from colossalai_amd import ops

    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "train":
        out = ops.qkv_norm_rope(s["qkv"], *s["weights"], s["table"], h, kv, positions=s["positions"], eps=1e-6)
        return list(out) + list(torch.autograd.grad(out, [s["qkv"], *s["weights"]], s["grads"]))
    if case["kind"] == "attend":
        return ops.paged_attention_4bit(s["q"], s["kpool"], s["vpool"], s["batch"], d ** -0.5, window=case["window"])
    q, k, v = s["qkv"].view(-1, h + 2 * kv, d).split([h, kv, kv], 1)
    wq, wk = s.get("weights", (None, None))
    q = ops.paged_kv_append(q, k, v, s["kpool"], s["vpool"], s["rows"], s["positions"], s["table"], wq, wk, eps=1e-6)
    if case["kind"] == "step":
        return ops.paged_attention_4bit(q, s["kpool"], s["vpool"], s["batch"], d ** -0.5, window=case["window"])
    if case["bits"] == 4:
        return q, *ops.kv4_read(s["kpool"], s["vpool"], s["rows"], d)
    return q, s["kpool"], s["vpool"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ the exact results
def _turn(x, table, positions, back=False):
    """The rotation of x [tokens, heads, D] in 64 bits, as a product of complex numbers; `back`: its transpose."""
    c, s = table.double()[positions.long()].chunk(2, -1)
    z = torch.complex(*(t.contiguous() for t in x.chunk(2, -1))) * torch.complex(c, -s if back else s)[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_train(s):
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    rows = case["batch"] * case["seq"]
    pos = torch.arange(rows, device="cuda") % case["seq"] if s["positions"] is None else s["positions"]
    x = s["qkv"].detach().double().view(rows, -1, d)
    out, dx, dws = [], torch.empty_like(x), []
    for lo, n, w, g in ((0, h, s["weights"][0], s["grads"][0]), (h, kv, s["weights"][1], s["grads"][1])):
        part, w = x[:, lo: lo + n], w.detach().double()
        size = (part.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt()
        unit = part / size
        out.append(_turn(unit * w, s["table"], pos).view(case["batch"], case["seq"], n, d))
        back = _turn(g.double().view(rows, n, d), s["table"], pos, True)
        dws.append((back * unit).sum((0, 1)))
        back = back * w
        dx[:, lo: lo + n] = (back - unit * (back * unit).sum(-1, keepdim=True) / d) / size
    out.append(x[:, h + kv:].reshape(case["batch"], case["seq"], kv, d))
    dx[:, h + kv:] = s["grads"][2].double().view(rows, kv, d)
    return out + [dx.view(case["batch"], case["seq"], -1), *dws]


def _exact_heads(s):
    """Queries and keys after norm and rotation, and values, in 64 bits."""
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    q, k = x[:, :h], x[:, h: h + kv]
    if "weights" in s:
        q, k = (t / (t.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double() for t, w in zip((q, k), s["weights"]))
    return _turn(q, s["table"], s["positions"]), _turn(k, s["table"], s["positions"]), x[:, h + kv:]


def _exact_4bit(x):
    """The nearest numbers of a 4-bit cache to x [tokens, heads, D] in 64 bits."""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2((most / 6).clamp(min=2.0 ** -126))))
    unit = torch.where(unit * 6 < most, unit * 2, torch.where((unit * 3 >= most) & (unit > 2.0 ** -126), unit / 2, unit))
    a = x.abs() / unit
    step = torch.where(a <= 2, 0.5, torch.where(a <= 4, 1.0, 2.0))  # the numbers' distance: half an even multiple is even
    return (torch.sign(x) * torch.round(a / step) * step * unit).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "train":
        return _exact_train(s)
    if kind != "attend":
        q, k, v = _exact_heads(s)
        if kind == "append" and case["bits"] == 4:
            return q, _exact_4bit(k), _exact_4bit(v)
        if kind == "append":
            pools = []
            for pool, x in ((s["kpool"], k), (s["vpool"], v)):
                pool = pool.double().flatten(0, 1)
                pool[s["rows"].long()] = x
                pools.append(pool.view(s["kpool"].shape))
            return q, *pools
    else:
        q = s["q"].double()
    counts, starts, tables, pages = _batch(case, seed)
    kv, d, ps = case["kv_heads"], case["dim"], case["page"]
    if sum(c * (c + b) for c, b in zip(counts, starts)) * case["heads"] * d > 2e12:
        return None
    codes = _cache(_gen(seed), case, pages)
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    out, at = [], 0
    for i, (n, b) in enumerate(zip(counts, starts)):
        pick = torch.tensor(tables[i], device="cuda")
        both = []
        for code, scale in (codes[:2], codes[2:]):
            code, scale = code[pick].flatten(0, 1)[: b + n], scale[pick].flatten(0, 1)[: b + n]
            both.append(grid[(code & 7).long()] * (1.0 - 2.0 * (code >> 3)) * torch.exp2(scale.double() - 127).repeat_interleave(32, -1))
        if kind == "step":
            both[0][b:], both[1][b:] = _exact_4bit(k[at: at + n]), _exact_4bit(v[at: at + n])
        mine, rows = [], torch.arange(b, b + n, device="cuda")[:, None]
        col = torch.arange(b + n, device="cuda")[None]
        hide = (col > rows) | ((rows - col >= case["window"]) if case["window"] else False)
        for head in range(case["heads"]):
            of = head // (case["heads"] // kv)
            w = q[at: at + n, head] @ both[0][:, of].t() / math.sqrt(d)
            mine.append(torch.softmax(w.masked_fill(hide, -math.inf), -1) @ both[1][:, of])
        out.append(torch.stack(mine, 1))
        at += n
    return torch.cat(out)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "train":
        rows, size = case["batch"] * case["seq"], 2 if case["dtype"] != "fp32" else 4
        # forward: the projection in, its parts out; backward: the projection and three gradients in, one out
        return {"bytes": (5.0 * (h + 2 * kv) - kv) * d * rows * size + 8.0 * d * case["seq"], "flops": 30.0 * rows * (h + kv) * d}
    if case["kind"] == "append":
        n = case["tokens"]
        out = 2 * kv * d * (17 / 32 if case["bits"] == 4 else 2)
        return {"bytes": n * ((h + 2 * kv) * d * 2 + h * d * 2 + out) + 4.0 * d * min(n, 8192), "flops": 12.0 * n * (h + kv) * d}
    # the lengths are drawn by the seed: their mean
    n, cached, window = 0, 0.0, case["window"] or 1 << 40
    counts, starts, _, _ = _batch(case, 1)
    n = sum(counts)
    cached = sum(min(b + c, window + c) for c, b in zip(counts, starts))
    pairs = sum(sum(min(p + 1, window) for p in range(b, b + c)) for c, b in zip(counts, starts))
    more = n * (h + 2 * kv) * d * 2 + 2 * kv * n * d * 17 / 32 if case["kind"] == "step" else 0
    return {"bytes": cached * kv * d * 2 * 17 / 32 + 4.0 * n * h * d + more, "flops": 4.0 * pairs * h * d}
