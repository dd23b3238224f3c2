"""``qkv_norm_rope``: a packed projection's heads split, normed and rotated, and the gradients, against the formulas in 64 bits.

Bounds. A result is rounded to its type once, at most ``eps / 2`` of it. Ahead of that, in float32: squares and their sum over D <= 512
channels (an exchange tree: at most 16 + 5 roundings deep), a mean, a root, three products and a turn: at most 32 roundings of 2^-24
of the row's largest value times sqrt(2): under 2^-18 of it. dx has another sum like it, and cancels: 2^-17 of the row's largest
|w dy| / rms. A weight's gradient sums over tokens and heads: a term has 2^-18, and each of the roundings of the sums
(tokens and heads of a wave one after the other, at most n, then a tree) at most 2^-24 of the sum of magnitudes."""

import pytest
import torch

from colossalai_amd.ops import build_rope_table, qkv_norm_rope

gpu = pytest.mark.gpu


def _turn(x, table, at, back=False):
    half = x.shape[-1] // 2
    c, s = table[at][..., None, :half], table[at][..., None, half:] * (-1 if back else 1)
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def _formula(qkv, wq, wk, table, H, G, at, eps, grads):
    """Outputs and gradients in 64 bits, and the sums of magnitudes of the weights' gradients."""
    B, S, D = *qkv.shape[:2], wq.numel()
    x, table = qkv.detach().double().view(B, S, -1, D), table.double()
    at = torch.arange(S, device=x.device).expand(B, S) if at is None else at.long().view(B, S)
    outs, dx, dws, sizes = [], [], [], []
    for part, w, g in ((x[:, :, :H], wq, grads[0]), (x[:, :, H:H + G], wk, grads[1])):
        w, rms = w.detach().double(), (part.square().mean(-1, keepdim=True) + eps).sqrt()
        u = part / rms
        outs.append(_turn(u * w, table, at))
        a = _turn(g.double(), table, at, back=True)
        dws.append((a * u).sum((0, 1, 2)))
        sizes.append((a * u).abs().sum((0, 1, 2)))
        a = a * w
        dx.append((a - u * (a * u).mean(-1, keepdim=True)) / rms)
        sizes.append((a / rms).abs().amax(-1, keepdim=True))
    outs.append(x[:, :, H + G:])
    return outs, torch.cat(dx + [grads[2].double()], 2), dws, sizes


def _inputs(B, S, H, G, D, dtype, wide, device, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    qkv = (torch.randn(B, S, (H + 2 * G) * D, generator=g) * torch.exp(torch.randn(B, S, 1, generator=g))).to(device, dtype)
    ws = [(1 + 0.3 * torch.randn(D, generator=g)).to(device, torch.float32 if wide else dtype) for _ in range(2)]
    grads = [torch.randn(B, S, n, D, generator=g).to(device, dtype) for n in (H, G, G)]
    return qkv, ws, grads


def _check(qkv, ws, grads, table, H, G, at, eps=1e-6):
    dtype, n = qkv.dtype, qkv.shape[0] * qkv.shape[1] * H
    leaves = [qkv.detach().requires_grad_(), *(w.detach().requires_grad_() for w in ws)]
    out = qkv_norm_rope(*leaves, table, H, G, positions=at, eps=eps)
    got = torch.autograd.grad(out, leaves, grads)
    want, dx, dws, sizes = _formula(qkv, *ws, table, H, G, at, eps, grads)
    half = torch.finfo(dtype).eps / 2
    tiny = 0 if dtype != torch.float16 else 2.0 ** -25  # half a step of the smallest numbers
    for o, y, g in zip(out[:2], want, (H, G)):
        assert o.shape == y.shape and o.dtype == dtype and o.is_contiguous()
        assert ((o.double() - y).abs() <= half * y.abs() + 2.0 ** -18 * y.abs().amax(-1, keepdim=True) * 1.42 + tiny).all()
    assert torch.equal(out[2].double(), want[2]) and out[2].is_contiguous()
    gx = got[0].double().view(dx.shape)
    assert torch.equal(gx[:, :, H + G:], dx[:, :, H + G:])
    size = torch.cat([sizes[1], sizes[3]], 2)
    assert ((gx - dx).abs()[:, :, :H + G] <= half * dx.abs()[:, :, :H + G] + 2.0 ** -17 * 1.42 * size + tiny).all()
    for a, b, s in zip(got[1:], dws, (sizes[0], sizes[2])):
        assert a.dtype == ws[0].dtype
        assert ((a.double() - b).abs() <= torch.finfo(a.dtype).eps / 2 * b.abs() + (2.0 ** -18 + n * 2.0 ** -24) * s + tiny).all()
    return out, got


SHAPES = [(1, 1, 1, 1, 16), (2, 7, 3, 1, 48), (1, 33, 4, 4, 64), (3, 50, 6, 2, 80), (2, 129, 8, 2, 96), (1, 300, 28, 4, 128), (2, 65, 5, 5, 256),
          (1, 9, 2, 1, 512), (1, 5000, 2, 2, 128)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,H,G,D", SHAPES)
def test_against_the_formula(B, S, H, G, D, dtype):
    qkv, ws, grads = _inputs(B, S, H, G, D, dtype, False, "cuda")
    _check(qkv, ws, grads, build_rope_table(max(S, 8), D, 1e4, "cuda"), H, G, None)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_positions_strides_and_wide_weights(dtype):
    """Positions in any order, rows that lie apart and at odd places, weights in float32, gradients that are views."""
    B, S, H, G, D = 2, 37, 4, 2, 64
    table = build_rope_table(500, D, 1e4, "cuda")
    at = torch.randint(0, 500, (B, S), generator=torch.Generator().manual_seed(3)).int().cuda()
    qkv, ws, grads = _inputs(B, S, H, G, D, dtype, True, "cuda")
    W = qkv.shape[2]
    _, want = _check(qkv, ws, grads, table, H, G, at)
    for lead, tail in ((8, 16), (3, 5)):  # multiples of 16 bytes, and not
        room = torch.full((S, B, lead + W + tail), 7.0, device="cuda", dtype=dtype)
        view = room[:, :, lead: lead + W].transpose(0, 1)
        view.copy_(qkv)
        wide = [torch.randn(*g.shape[:3], 3 * D, device="cuda").to(dtype) for g in grads]
        for a, g in zip(wide, grads):
            a[..., 1: D + 1] = g
        _, got = _check(view, ws, [a[..., 1: D + 1] for a in wide], table, H, G, at)
        assert all(torch.equal(a.reshape(-1), b.reshape(-1)) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_and_tables_at_any_address(dtype):
    qkv, ws, grads = _inputs(2, 40, 3, 1, 64, dtype, dtype == torch.float32, "cuda")
    table = build_rope_table(64, 64).cuda()
    apart = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    _check(qkv, [apart(w) for w in ws], grads, apart(table), 3, 1, None)


@gpu
def test_small_large_and_not_finite_rows():
    """Rows of zeros and of numbers whose squares vanish beside eps; a NaN stays in its head; positions that the table does not have."""
    B, S, H, G, D = 1, 12, 2, 1, 64
    table = build_rope_table(S, D, 1e4, "cuda")
    qkv, ws, grads = _inputs(B, S, H, G, D, torch.float32, False, "cuda")
    qkv[0, 0] = 0
    qkv[0, 1] *= 1e-6
    qkv[0, 2] *= 1e15
    _check(qkv, ws, grads, table, H, G, None)
    clean = qkv_norm_rope(qkv, *ws, table, H, G)
    bad = qkv.clone()
    bad[0, 5, 3] = float("nan")
    got = qkv_norm_rope(bad, *ws, table, H, G)
    assert got[0][0, 5, 0].isnan().all()
    got[0][0, 5, 0] = clean[0][0, 5, 0]
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    at = torch.arange(S, device="cuda").int()
    at[4], at[7] = -1, S
    got = qkv_norm_rope(qkv, *ws, table, H, G, positions=at)
    assert all(t[0, i].isnan().all() for t in got[:2] for i in (4, 7))
    assert all(torch.equal(a[0, 8:], b[0, 8:]) for a, b in zip(got, clean)) and torch.equal(got[2], clean[2])


@gpu
def test_no_tokens():
    qkv = torch.zeros(2, 0, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ws = [torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2)]
    out = qkv_norm_rope(qkv, *ws, build_rope_table(8, 64, 1e4, "cuda"), 2, 1)
    assert [tuple(t.shape) for t in out] == [(2, 0, 2, 64), (2, 0, 1, 64), (2, 0, 1, 64)]
    got = torch.autograd.grad(out, [qkv, *ws], [torch.zeros_like(t) for t in out])
    assert got[0].shape == qkv.shape and not got[1].any() and not got[2].any()


@gpu
def test_gradient_against_differences():
    """A directional difference with step h = 2^-6: its own error is h^2 / 6 of a third derivative, here under 2^-8 of the gradient's length
    times the direction's, and float32 outputs add 2^-24 * |outputs| * |dy| / h."""
    B, S, H, G, D, h = 1, 6, 2, 1, 64, 2.0 ** -6
    table = build_rope_table(S, D, 1e4, "cuda")
    qkv, ws, grads = _inputs(B, S, H, G, D, torch.float32, False, "cuda")
    leaves = [t.detach().requires_grad_() for t in (qkv, *ws)]
    got = torch.autograd.grad(qkv_norm_rope(*leaves, table, H, G), leaves, grads)
    of = lambda *a: sum((o.double() * g.double()).sum() for o, g in zip(qkv_norm_rope(*a, table, H, G), grads))  # noqa: E731
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        d /= d.norm()
        up, down = ([t.detach() + (s * h * d if j == i else 0) for j, t in enumerate(leaves)] for s in (1, -1))
        slope = (of(*up) - of(*down)) / (2 * h)
        size = got[i].double().norm() + 2.0 ** -24 / h * sum(g.double().norm() for g in grads) * 30
        assert (slope - (got[i].double() * d).sum()).abs() <= 2.0 ** -8 * size


@gpu
def test_gradients_of_gradients_and_unused_parts():
    B, S, H, G, D = 1, 5, 2, 1, 32
    table = build_rope_table(S, D, 1e4, "cuda")
    qkv, ws, grads = _inputs(B, S, H, G, D, torch.float32, False, "cuda")
    leaves = [t.detach().requires_grad_() for t in (qkv, *ws)]
    out = qkv_norm_rope(*leaves, table, H, G)
    first = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    again = torch.autograd.grad(out, leaves, grads, create_graph=True)
    for a, b in zip(first, again):
        assert ((a - b).abs() <= 2.0 ** -17 * b.abs().amax() * 8).all()  # two orders of float32 sums
    assert torch.autograd.grad(again[0].square().sum(), leaves[0])[0].isfinite().all()
    q = qkv_norm_rope(*leaves, table, H, G)[0]
    got = torch.autograd.grad(q, leaves, grads[0])
    assert not got[0].view(S, -1, D)[:, H:].any() and not got[2].any() and got[1].any()
    plain = qkv_norm_rope(leaves[0], ws[0], ws[1], table, H, G)
    torch.autograd.grad(plain, leaves[0], grads)


EACH = ["cpu", pytest.param("cuda", marks=gpu)]


def _derivatives(of, leaves, grads, by):
    """Gradients of ``leaves`` by ``grads``, and of their product with ``by`` the gradients of all of them."""
    leaves, grads = ([t.detach().requires_grad_() for t in ts] for ts in (leaves, grads))
    first = torch.autograd.grad(of(*leaves), leaves, grads, create_graph=True)
    return first, torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, by)), [*leaves, *grads])


@pytest.mark.parametrize("device", EACH)
@pytest.mark.parametrize("placed", [False, True])
def test_second_derivatives(placed, device):
    """Against those of the formula in 64 bits. A float32 number has at most D + 32 < 2^7 roundings behind it, each 2^-24 of a term that is at most
    2^3 times the tensor's largest number (nothing cancels further in random rows of one size): 2^-14 of that."""
    B, S, H, G, D = 2, 7, 3, 2, 64
    g = torch.Generator().manual_seed(4)
    leaves = [torch.randn(B, S, (H + 2 * G) * D, generator=g), *(1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))]
    by = [torch.randn(t.shape, generator=g).to(device) for t in leaves]
    grads = [torch.randn(B, S, n, D, generator=g).to(device) for n in (H, G, G)]
    leaves, table = [t.to(device) for t in leaves], build_rope_table(40, D, 1e4, device)
    at = torch.randint(0, 40, (B, S), generator=g).int().to(device) if placed else None

    def formula(qkv, wq, wk):
        q, k, v = qkv.view(B, S, -1, D).split([H, G, G], 2)
        place = torch.arange(S, device=device).expand(B, S) if at is None else at.long()
        norm = lambda x, w: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
        return [_turn(norm(q, wq), table.double(), place), _turn(norm(k, wk), table.double(), place), v]

    got = _derivatives(lambda *t: qkv_norm_rope(*t, table, H, G, positions=at), leaves, grads, by)
    want = _derivatives(formula, *([t.double() for t in ts] for ts in (leaves, grads, by)))
    for a, b in zip([*got[0], *got[1]], [*want[0], *want[1]]):
        assert a.dtype == torch.float32 and ((a.double() - b).abs() <= 2.0 ** -14 * b.abs().amax()).all()


@pytest.mark.parametrize("device", EACH)
def test_second_derivatives_at_positions_that_the_table_does_not_have(device):
    """They are NaN for those tokens' queries and keys, and what they are for all others."""
    B, S, H, G, D = 1, 12, 2, 1, 32
    table = build_rope_table(S, D, 1e4, device)
    qkv, ws, grads = _inputs(B, S, H, G, D, torch.float32, False, device)
    by = [torch.ones_like(t) for t in (qkv, *ws)]
    by[1].zero_(), by[2].zero_()  # the weights' gradients are sums over all tokens
    at = torch.arange(S, device=device).int()
    want = _derivatives(lambda *t: qkv_norm_rope(*t, table, H, G, positions=at), [qkv, *ws], grads, by)
    lost = at.clone()
    lost[2], lost[5], lost[9] = -1, S, 2 ** 31 - 1
    got = _derivatives(lambda *t: qkv_norm_rope(*t, table, H, G, positions=lost), [qkv, *ws], grads, by)
    held = torch.tensor([i not in (2, 5, 9) for i in range(S)], device=device)
    for a, b in ((got[0][0], want[0][0]), (got[1][0], want[1][0]), (got[1][3], want[1][3])):
        a, b = (t.reshape(S, -1, D) for t in (a, b))
        assert torch.equal(a[held], b[held])
    for a in (got[0][0], got[1][0]):
        a = a.view(S, -1, D)[~held]
        assert a[:, : H + G].isnan().all() and not a[:, H + G:].isnan().any()
    none = qkv_norm_rope(qkv, *ws, table[:0], H, G, positions=at)  # a table of no rows has no position
    assert none[0].isnan().all() and none[1].isnan().all() and torch.equal(none[2], qkv.view(B, S, -1, D)[:, :, H + G:])
    first, second = _derivatives(lambda *t: qkv_norm_rope(*t, table[:0], H, G, positions=at), [qkv, *ws], grads, by)
    assert first[0].view(S, -1, D)[:, : H + G].isnan().all() and second[0].view(S, -1, D)[:, : H + G].isnan().all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_that_are_broadcast(dtype):
    """Gradients of one value for all channels, heads or tokens, as sums leave them."""
    B, S, H, G, D = 2, 21, 4, 2, 64
    qkv, ws, grads = _inputs(B, S, H, G, D, dtype, False, "cuda")
    spread = [grads[0][:1, :1, :1, :1].expand_as(grads[0]), grads[1][:, :, :1].expand_as(grads[1]), grads[2][:1].expand_as(grads[2])]
    _check(qkv, ws, spread, build_rope_table(S, D, 1e4, "cuda"), H, G, None)


@gpu
def test_another_stream_and_a_captured_graph():
    B, S, H, G, D = 2, 64, 4, 2, 64
    table = build_rope_table(S, D, 1e4, "cuda")
    qkv, ws, grads = _inputs(B, S, H, G, D, torch.bfloat16, False, "cuda")

    def step():
        leaves = [t.detach().requires_grad_() for t in (qkv, *ws)]
        out = qkv_norm_rope(*leaves, table, H, G)
        return [*out, *torch.autograd.grad(out, leaves, grads)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for scale in (2.0, 0.5, 1.0):
        qkv.mul_(scale)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refusals():
    table, w = build_rope_table(16, 32), torch.ones(32)
    x = torch.zeros(1, 8, 4 * 32)
    for bad in (dict(qkv=x[0]), dict(qkv=x.double()), dict(qkv=x.long()), dict(q_weight=torch.ones(24), k_weight=torch.ones(24)), dict(k_weight=torch.ones(16)),
                dict(q_weight=w.half()), dict(q_weight=w.bfloat16(), k_weight=w.bfloat16()), dict(num_heads=3), dict(num_kv_heads=0),
                dict(table=table.double()), dict(table=table[:, :16]), dict(table=table[:4]), dict(positions=torch.arange(8)),
                dict(positions=torch.arange(7).int())):
        args = dict(qkv=x, q_weight=w, k_weight=w, table=table, num_heads=2, num_kv_heads=1) | bad
        with pytest.raises(ValueError):
            qkv_norm_rope(**args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_on_the_cpu(dtype):
    qkv, ws, grads = _inputs(2, 9, 4, 2, 32, dtype, True, "cpu")
    _check(qkv, ws, grads, build_rope_table(16, 32), 4, 2, None)
    at = torch.arange(18).int().flip(0) % 16
    _check(qkv, ws, grads, build_rope_table(16, 32), 4, 2, at)
