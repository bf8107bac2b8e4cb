"""Rotary positions, head norms and paged appends on the GPU, against float64."""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from heads_util import E, close, half_eps, make_batch, partner_abs, tiny, turn_bound
from oracle import heads as oracle

pytestmark = gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def randn(g, *shape):
    return torch.randn(*shape, generator=g)


# lead, q heads, k heads, dim, rotary, interleaved, layout of the inputs
SHAPES = [
    ((3, 5), 4, 2, 64, 64, False, "dense"),
    ((1,), 1, 1, 128, 128, True, "dense"),
    ((2, 7), 6, 2, 128, 64, False, "fused"),
    ((257,), 3, 1, 80, 48, True, "fused"),
    ((2, 3), 2, 2, 256, 256, False, "bhsd"),
    ((4, 1), 5, 5, 72, 72, False, "dense"),       # halves off the vectors
    ((11,), 2, 1, 66, 22, True, "dense"),         # rows off the vectors
    ((2, 2, 3), 2, 1, 96, 32, False, "dense"),
    ((9,), 2, 3, 2, 2, False, "dense"),           # the smallest head
    ((5,), 1, 2, 200, 8, True, "offset"),         # one element off the alignment
    ((3,), 2, 1, 1030, 514, False, "dense"),      # more than a wave's vectors
    ((0,), 4, 2, 64, 64, False, "dense"),
    ((2, 6), 4, 2, 64, 64, True, "expanded"),
    ((3, 5), 4, 2, 128, 56, False, "fused"),      # halves on 8 bytes,
    ((37,), 2, 2, 128, 44, True, "dense"),        # on 4,
    ((130,), 3, 1, 72, 36, False, "dense"),
    ((7,), 2, 1, 256, 12, False, "bhsd2"),
]


def make(g, lead, heads, dim, dtype, layout):
    """A tensor [*lead, heads, dim] on the GPU in the given layout."""
    if layout == "fused":
        return randn(g, *lead, heads + 3, dim).to(dtype).to(DEV)[..., 2:2 + heads, :]
    if layout == "bhsd":
        return randn(g, lead[0], heads, lead[1], dim).to(dtype).to(DEV).transpose(1, 2)
    if layout == "bhsd2":
        return randn(g, heads, *lead, dim).to(dtype).to(DEV).movedim(0, -2)
    if layout == "offset":
        n = math.prod(lead) * heads * dim
        return randn(g, n + 1).to(dtype).to(DEV)[1:].view(*lead, heads, dim)
    if layout == "expanded":
        return randn(g, *lead[:-1], 1, heads, dim).to(dtype).to(DEV).expand(*lead, heads, dim)
    return randn(g, *lead, heads, dim).to(dtype).to(DEV)


def flat(x):
    return x.detach().cpu().reshape(-1, *x.shape[-2:])


def table_of(rotary, n, factor=1.0):
    from kernels.hip.rotary import rotary_table
    return rotary_table(rotary, n, attention_factor=factor)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_rotary(case, dtype):
    need_gpu()
    from kernels.hip import rotary
    lead, hq, hk, dim, rot, inter, layout = case
    say("rotary", case, dtype)
    g = torch.Generator().manual_seed(1)
    q, k = make(g, lead, hq, dim, dtype, layout), make(g, lead, hk, dim, dtype, layout)
    gq, gk = make(g, lead, hq, dim, dtype, layout), make(g, lead, hk, dim, dtype, layout)
    table = table_of(rot, 5000, 1.1)
    pos = torch.randint(0, 5000, lead, generator=g)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = rotary.kernel_fn(q, k, table.to(DEV), pos.to(DEV), interleaved=inter)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    cos, sin = oracle.from_table(table, pos.reshape(-1))
    for x, y, up, dx in ((q, yq, gq, dq), (k, yk, gk, dk)):
        assert y.shape == x.shape and y.is_contiguous() and y.dtype == dtype and dx.shape == x.shape
        want = oracle.turn(flat(x), cos, sin, inter)
        close(flat(y), want, turn_bound(want, flat(x), rot, inter, dtype, factor=1.1), "forward")
        want = oracle.turn(flat(up), cos, -sin, inter)
        close(flat(dx), want, turn_bound(want, flat(up), rot, inter, dtype, factor=1.1), "backward")


def test_rotary_positions_far_and_wide():
    """Tables of far positions against angles in float64; None, int32, broadcast and per-sequence positions."""
    need_gpu()
    from kernels.hip import rotary
    g = torch.Generator().manual_seed(2)
    n, dim = 600001, 64
    table = rotary.rotary_table(dim, n, device=DEV)
    q = randn(g, 2, 5, 3, dim).to(DEV)
    pos = torch.tensor([[n - 1, 0, 262144, 1, 131071], [5, 524288, 65537, n - 2, 99999]])
    say("far positions")
    y, none = rotary.kernel_fn(q, None, table, pos.to(DEV))
    assert none is None
    a = oracle.angles(pos.reshape(-1), dim)
    want = oracle.turn(flat(q), a.cos(), a.sin())
    close(flat(y), want, turn_bound(want, flat(q), dim, False, torch.float32), "far")
    assert torch.equal(rotary.kernel_fn(q, None, table, pos.int().to(DEV))[0], y)
    counted = rotary.kernel_fn(q, None, table)[0]
    row = torch.arange(5, device=DEV)
    for p in (row, row.expand(2, 5), row[None]):
        assert torch.equal(rotary.kernel_fn(q, None, table, p)[0], counted)
    col = torch.tensor([[7], [9]], device=DEV)
    assert torch.equal(rotary.kernel_fn(q, None, table, col)[0], rotary.kernel_fn(q, None, table, col.expand(2, 5))[0])
    one = rotary.kernel_fn(q[0, 0], None, table, torch.tensor(3, device=DEV))[0]
    assert torch.equal(one, rotary.kernel_fn(q[:1, :1], None, table, torch.tensor([[3]], device=DEV))[0][0, 0])
    assert torch.equal(rotary.kernel_fn(q[0, 0], None, table)[0], q[0, 0])  # position 0


def test_rotary_outside_the_table_is_nan():
    need_gpu()
    from kernels.hip import rotary
    g = torch.Generator().manual_seed(3)
    for dim, rot in ((64, 32), (66, 30)):
        q = randn(g, 4, 2, dim).to(DEV)
        table = table_of(rot, 10).to(DEV)
        pos = torch.tensor([-1, 9, 10, 2 ** 40], device=DEV)
        say("outside the table", dim)
        y, _ = rotary.kernel_fn(q, None, table, pos)
        assert torch.isnan(y[[0, 2, 3], :, :rot]).all() and torch.isfinite(y[1]).all()
        assert torch.equal(y[..., rot:], q[..., rot:])


def test_rotary_is_differentiable_again():
    need_gpu()
    from kernels.hip import rotary
    g = torch.Generator().manual_seed(4)
    q, k = randn(g, 6, 2, 64).to(DEV).requires_grad_(), randn(g, 6, 1, 64).to(DEV).requires_grad_()
    table = table_of(64, 6).to(DEV)
    say("second derivative")
    yq, yk = rotary.kernel_fn(q, k, table)
    # d/dq of (y^2).sum() / 2 is q (the turn keeps lengths), its derivative along v is v
    (gq, gk) = torch.autograd.grad((yq.square().sum() + yk.square().sum()) / 2, (q, k), create_graph=True)
    close(gq.detach(), q.detach().double().cpu(), 8 * E * partner_abs(q.detach().cpu(), 64, False), "first")
    v = randn(g, 6, 2, 64).to(DEV)
    (hv,) = torch.autograd.grad((gq * v).sum(), q)
    close(hv, v.double().cpu(), 16 * E * partner_abs(v.cpu(), 64, False), "second")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("turned", [True, False])
@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_norm(case, turned, dtype):
    need_gpu()
    from kernels.hip import qk_norm_rotary
    lead, hq, hk, dim, rot, inter, layout = case
    say("norm", case, turned, dtype)
    g = torch.Generator().manual_seed(5)
    eps = 1e-5
    q, k = make(g, lead, hq, dim, dtype, layout), make(g, lead, hk, dim, dtype, layout)
    gq, gk = make(g, lead, hq, dim, dtype, layout), make(g, lead, hk, dim, dtype, layout)
    wq, wk = (1 + 0.3 * randn(g, dim)).to(dtype).to(DEV), (1 + 0.3 * randn(g, dim)).to(dtype).to(DEV)
    table = table_of(rot, 5000) if turned else None
    pos = torch.randint(0, 5000, lead, generator=g) if turned else None
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rotary.kernel_fn(*leaves, table.to(DEV) if turned else None, pos.to(DEV) if turned else None, eps=eps,
                                      interleaved=inter)
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    p = pos.reshape(-1) if turned else None
    r = rot if turned else 0
    for x, w, y, up, dx, dw in ((q, wq, yq, gq, grads[0], grads[2]), (k, wk, yk, gk, grads[1], grads[3])):
        x, w, up = flat(x), w.cpu(), flat(up)
        z = oracle.norm(x, w, eps)
        want = oracle.norm_turn(x, w, eps, table, p, inter)
        close(flat(y), want, turn_bound(want, z, r, inter, dtype, units=51.0), "forward")
        wx, ww = oracle.norm_turn_grad(x, w, eps, table, p, up, inter)
        rms = torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
        n = x.double() / rms
        dz = partner_abs(up, r, inter)
        gw = dz * w.double().abs()
        bound = half_eps(dtype) * wx.abs() + 150 * E * (gw + n.abs() * (gw * n.abs()).mean(-1, keepdim=True)) / rms
        close(flat(dx), wx, bound + tiny(dtype), "dx")
        # chains: rows of a thread, the workgroup's row slots, the workgroups by eights
        rows = x.shape[0] * x.shape[1]
        chain = rows / 1024 + 1 + 256 + 128 + 8 + 60
        close(dw, ww, half_eps(dtype) * ww.abs() + chain * E * (dz * n.abs()).sum((0, 1)) + tiny(dtype), "dweight")


def test_norm_many_rows():
    """More rows than a workgroup each: the weights' gradients of 40000 heads."""
    need_gpu()
    from kernels.hip import qk_norm_rotary
    g = torch.Generator().manual_seed(6)
    tokens, hq, hk, dim = 5001, 7, 1, 128
    table = table_of(dim, tokens)
    leaves = [t.to(DEV).requires_grad_() for t in (randn(g, tokens, hq, dim), randn(g, tokens, hk, dim), 1 + 0.1 * randn(g, dim),
                                                   1 + 0.1 * randn(g, dim))]
    up = randn(g, tokens, hq, dim).to(DEV), randn(g, tokens, hk, dim).to(DEV)
    say("many rows")
    out = qk_norm_rotary.kernel_fn(*leaves, table.to(DEV))
    grads = torch.autograd.grad(out, leaves, up)
    for i in (0, 1):
        x, w, u = leaves[i].detach().cpu(), leaves[2 + i].detach().cpu(), up[i].cpu()
        dx, dw = oracle.norm_turn_grad(x, w, 1e-6, table, torch.arange(tokens), u)
        n = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True))
        mass = (partner_abs(u, dim, False) * n.abs()).sum((0, 1))
        close(grads[2 + i], dw, (tokens * hq / 1024 + 453) * E * mass, "dweight")
    again = torch.autograd.grad(qk_norm_rotary.kernel_fn(*leaves, table.to(DEV)), leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_norm_gradient_against_differences():
    need_gpu()
    from kernels.hip import qk_norm_rotary
    g = torch.Generator().manual_seed(7)
    x = [randn(g, 3, 2, 64), randn(g, 3, 1, 64), 1 + 0.2 * randn(g, 64), 1 + 0.2 * randn(g, 64)]
    up = [randn(g, 3, 2, 64), randn(g, 3, 1, 64)]
    table = table_of(32, 3)
    leaves = [t.to(DEV).requires_grad_() for t in x]
    say("differences")
    grads = torch.autograd.grad(qk_norm_rotary.kernel_fn(*leaves, table.to(DEV)), leaves, [u.to(DEV) for u in up])

    def value(a):
        pos = torch.arange(3)
        return sum(float((oracle.norm_turn(a[i], a[2 + i], 1e-6, table, pos) * up[i].double()).sum()) for i in (0, 1))

    h = 1e-4  # the third derivative's h^2 and the rounding of float64 over h both below 1e-6
    for i, t in enumerate(x):
        d = randn(g, *t.shape).double()
        a = [y.double() for y in x]
        a[i] = x[i].double() + h * d
        hi = value(a)
        a[i] = x[i].double() - h * d
        want = (hi - value(a)) / (2 * h)
        assert abs(float((grads[i].double().cpu() * d).sum()) - want) <= 1e-4 * (1 + abs(want))


def test_norm_edges():
    """A zero head, an expanded upstream gradient, weights of another type, one tensor alone, only some gradients."""
    need_gpu()
    from kernels.hip import qk_norm_rotary
    g = torch.Generator().manual_seed(8)
    q = randn(g, 4, 2, 64)
    q[1, 0] = 0.0
    w = (1 + 0.1 * randn(g, 64)).to(DEV).requires_grad_()
    x = q.bfloat16().to(DEV).requires_grad_()
    say("norm edges")
    y, none = qk_norm_rotary.kernel_fn(x, None, w, None)
    assert none is None and (y[1, 0] == 0).all()
    y.sum().backward()
    wx, ww = oracle.norm_turn_grad(x.detach().cpu(), w.detach().cpu().bfloat16(), 1e-6, None, None, torch.ones(4, 2, 64))
    assert w.grad.dtype == torch.float32 and torch.isfinite(x.grad).all()
    close(w.grad, ww, half_eps(torch.bfloat16) * ww.abs() + 500 * E * 8, "weight of another type")
    (only,) = torch.autograd.grad(qk_norm_rotary.kernel_fn(x, None, w.detach(), None)[0].sum(), x)
    assert torch.equal(only, x.grad)
    (only,) = torch.autograd.grad(qk_norm_rotary.kernel_fn(x.detach(), None, w, None)[0].sum(), w)
    assert torch.equal(only, w.grad)
    k = randn(g, 4, 1, 64).bfloat16().to(DEV).requires_grad_()
    yq, yk = qk_norm_rotary.kernel_fn(x, k, w, w.detach())
    gq, gk = torch.autograd.grad(yq.sum(), (x, k))  # nothing reaches k
    assert torch.equal(gq, x.grad) and not gk.any()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(qk_norm_rotary.kernel_fn(x, None, w, None)[0].float().square().sum(), x, create_graph=True)


# ---------------------------------------------------------------------------
# Appends
# ---------------------------------------------------------------------------
# counts, lengths, page, q heads, k heads, dim, rotary, interleaved, normed
BATCHES = [
    ([1, 1, 1], [1, 17, 64], 16, 4, 2, 64, 64, False, False),
    ([5, 0, 3, 1], [5, 9, 30, 8], 8, 6, 2, 128, 64, False, True),
    ([33], [40], 1, 1, 1, 64, 64, True, False),
    ([2, 2], [70, 3], 48, 2, 1, 80, 16, True, True),
    ([4, 1], [4, 100], 7, 2, 2, 66, 66, False, True),
    ([3, 2], [2, 9], 4, 2, 1, 64, 32, False, False),     # a sequence shorter than its new tokens
    ([70] + [1] * 69, [70] + list(range(1, 70)), 16, 2, 1, 64, 64, False, True),
    ([21, 1], [30, 8], 16, 4, 2, 72, 36, False, True),   # halves on 4 bytes
    ([21, 1], [30, 8], 16, 4, 2, 128, 56, True, False),  # on 8
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", BATCHES, ids=lambda c: str(c[2:]))
def test_append(case, dtype):
    need_gpu()
    from kernels.hip import paged_append
    counts, lengths, page, hq, hk, dim, rot, inter, normed = case
    say("append", case, dtype)
    g = torch.Generator().manual_seed(9)
    pages, lens, starts, total = make_batch(counts, lengths, page, 10)
    tokens = sum(counts) + 3  # rows behind the last sequence
    qkv = randn(g, tokens, hq + 2 * hk, dim).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    kc, vc = randn(g, total, hk, page, dim).to(dtype), randn(g, total, page, hk, dim).to(dtype)
    wq, wk = (1 + 0.3 * randn(g, dim)).to(dtype), (1 + 0.3 * randn(g, dim)).to(dtype)
    table = table_of(rot, max(lengths) + 1)
    want_q, want_k, want_v = oracle.append(q, k, v, kc.transpose(1, 2), vc, pages, lens, starts, wq if normed else None,
                                           wk if normed else None, 1e-6, table, inter)
    dqkv, dkc, dvc = qkv.to(DEV), kc.to(DEV).transpose(1, 2), vc.to(DEV)
    args = (dqkv[:, hq:hq + hk], dqkv[:, hq + hk:], dkc, dvc, pages.to(DEV), lens.to(DEV), starts.to(DEV))
    kw = dict(table=table.to(DEV), interleaved=inter)
    if normed:
        kw.update(q_weight=wq.to(DEV), k_weight=wk.to(DEV))
    out = paged_append.kernel_fn(*args, q=dqkv[:, :hq], **kw)
    # what a token's key and its norm are, at its place
    units = 51.0 if normed else 4.0
    zk = oracle.norm(k, wk, 1e-6) if normed else k
    zq = oracle.norm(q, wq, 1e-6) if normed else q
    size = oracle.append(None, partner_abs(zk, rot, inter).abs(), v, torch.zeros_like(want_k), vc, pages, lens, starts, None,
                         None, 0.0, None, False)[1]
    close(dkc, want_k, half_eps(dtype) * want_k.abs() * (size > 0) + units * E * size + tiny(dtype) * (size > 0), "k_cache")
    assert torch.equal(dvc.cpu().double(), want_v)
    n = sum(counts)
    close(out[:n], want_q[:n], turn_bound(want_q[:n], zq[:n], rot, inter, dtype, units), "q")
    assert not out[n:].any()
    # in place, rows of no sequence as they were; the same places again
    keep = dqkv[n:, :hq].clone()
    inside = dqkv[:, :hq]
    before = dkc.clone()
    assert paged_append.kernel_fn(*args, q=inside, q_out=inside, **kw) is inside
    # (a token before its sequence has no angles: NaN)
    assert torch.equal(inside[:n].nan_to_num(9.0), out[:n].nan_to_num(9.0))
    assert torch.equal(inside[n:], keep) and torch.equal(dkc, before)


def test_append_without_queries_or_angles():
    need_gpu()
    from kernels.hip import paged_append
    g = torch.Generator().manual_seed(11)
    pages, lens, _, total = make_batch([2, 2, 2], [5, 2, 8], 4, 12)
    k, v = randn(g, 6, 2, 64).to(DEV), randn(g, 6, 2, 64).to(DEV)
    kc, vc = torch.zeros(total, 4, 2, 64, device=DEV), torch.zeros(total, 4, 2, 64, device=DEV)
    say("append alone")
    version = kc._version
    assert paged_append.kernel_fn(k, v, kc, vc, pages.to(DEV), lens.to(DEV)) is None
    assert kc._version > version
    for b, n in enumerate(lens.tolist()):
        for i in (0, 1):
            p = n - 2 + i
            at = int(pages[b, p // 4]), p % 4
            assert torch.equal(kc[at], k[2 * b + i]) and torch.equal(vc[at], v[2 * b + i])
    assert int((kc != 0).any(-1).sum()) == 12


def test_append_bad_pages_write_nothing():
    """Pages outside the cache, lengths past the table's width or negative, starts out of range or order."""
    need_gpu()
    from kernels.hip import paged_append
    g = torch.Generator().manual_seed(13)
    k, v = randn(g, 4, 1, 64).to(DEV), randn(g, 4, 1, 64).to(DEV)
    pages = torch.tensor([[9, 1], [-1, 0], [0, 2 ** 31 - 1], [-2 ** 31, 1]], dtype=torch.int32)
    say("append bad pages")
    for lengths, starts in (([3, 3, 7, 2], None), ([9, -5, 2 ** 31 - 1, -2 ** 31], None),
                            ([1, 1, 1, 1], [5, 9, -3, 100, 2 ** 31 - 1]), ([8, 8, 8, 8], [3, 2, 1, 0, -1])):
        kc, vc = torch.zeros(2, 4, 1, 64, device=DEV), torch.zeros(2, 4, 1, 64, device=DEV)
        st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV)
        paged_append.kernel_fn(k, v, kc, vc, pages.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), st, q=k,
                               table=table_of(64, 4).to(DEV))
        assert torch.isfinite(kc).all() or starts is not None
        if lengths[0] != 1 and starts is None:
            assert not vc.any()


def test_streams_and_graphs():
    """On another stream, and captured forward, backward and append replayed with new inputs."""
    need_gpu()
    from kernels.hip import paged_append, qk_norm_rotary, rotary
    g = torch.Generator().manual_seed(14)
    q, k = randn(g, 50, 4, 64).bfloat16().to(DEV), randn(g, 50, 2, 64).bfloat16().to(DEV)
    up = [randn(g, 50, 4, 64).bfloat16().to(DEV), randn(g, 50, 2, 64).bfloat16().to(DEV)]
    w = [(1 + 0.1 * randn(g, 64)).bfloat16().to(DEV) for _ in range(2)]
    table = table_of(64, 64).to(DEV)
    pages, lens, starts, total = make_batch([20, 30], [33, 30], 16, 15)
    pages, lens, starts = pages.to(DEV), lens.to(DEV), starts.to(DEV)
    kc = torch.zeros(total, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)

    def step():
        a, b = q.detach().requires_grad_(), k.detach().requires_grad_()
        c, d = w[0].detach().requires_grad_(), w[1].detach().requires_grad_()
        y = qk_norm_rotary.kernel_fn(a, b, c, d, table)
        grads = torch.autograd.grad(y, (a, b, c, d), up)
        z = rotary.kernel_fn(q, k, table, interleaved=True)
        r = paged_append.kernel_fn(k, k, kc, vc, pages, lens, starts, q=q, table=table)
        return [*(t.detach() for t in y), *grads, *z, r, kc, vc]

    say("eager")
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    say("capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        q.mul_(-1.5 if i else 1.0)
        up[0].add_(0.25)
        kc.zero_()
        want = [t.clone() for t in step()]
        for t in outs:
            t.fill_(7.0)
        torch.cuda.synchronize()
        say("replay", i)
        graph.replay()
        torch.cuda.synchronize()
        # the caches keep 7 in the places that no token has
        for j, (a, b) in enumerate(zip(outs, want)):
            if j >= len(outs) - 2:
                a, b = a[b.abs().sum(-1) > 0], b[b.abs().sum(-1) > 0]
            assert torch.equal(a, b), (i, j)


def test_more_rows_than_a_grid():
    """Past 2^20 workgroups' rows: positions 0 leave the heads as they are, others turn them."""
    need_gpu()
    from kernels.hip import rotary
    n = 2 ** 22 + 9  # (four a workgroup)
    say("many rows", n)
    x = randn(torch.Generator().manual_seed(2), n, 1, 2).to(torch.bfloat16).to(DEV)
    at = torch.zeros(n, dtype=torch.int32, device=DEV)
    at[-3:] = 1
    y = rotary.kernel_fn(x, None, table_of(2, 2).to(DEV), at)[0]
    assert torch.equal(y[:-3], x[:-3])
    want = oracle.turn(flat(x[-3:]), *oracle.from_table(table_of(2, 2), torch.ones(3, dtype=torch.long)))
    close(flat(y[-3:]), want, turn_bound(want, flat(x[-3:]), 2, False, torch.bfloat16))


def test_strides_past_32_bits():
    """Two tokens 2^32 + 8 elements apart, forward and back, against the same ones side by side."""
    need_gpu()
    from kernels.hip import qk_norm_rotary, rotary
    say("far strides")
    g = torch.Generator().manual_seed(3)
    near = randn(g, 2, 1, 64).to(torch.bfloat16).to(DEV)
    room = torch.empty(2 ** 32 + 8 + 64, dtype=torch.bfloat16, device=DEV)
    far = room.as_strided((2, 1, 64), (2 ** 32 + 8, 64, 1))
    far.copy_(near)
    w, table = (1 + 0.1 * randn(g, 64)).to(torch.bfloat16).to(DEV), table_of(64, 2).to(DEV)
    assert torch.equal(rotary.kernel_fn(far, None, table)[0], rotary.kernel_fn(near, None, table)[0])
    grads = []
    for x in (far, near):
        x, w1 = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = qk_norm_rotary.kernel_fn(x, None, w1, None, table)[0]
        grads.append([y.detach(), *torch.autograd.grad(y, (x, w1), x.detach())])
    # (their sums are taken in another order: both are half a step from sums of up to 64 products
    # of at most 32, a rounding in fp32 each)
    for a, b in zip(*grads):
        close(a, b.cpu(), 2.1 * half_eps(torch.bfloat16) * b.cpu().double().abs() + 2 * 64 * 32 * E)


def test_the_same_tensor_twice():
    """One tensor as queries and keys, one weight for both: the gradients are the sums; one cache for both is refused."""
    need_gpu()
    from kernels.hip import paged_append, qk_norm_rotary, rotary
    say("twice")
    g = torch.Generator().manual_seed(31)
    x, w = randn(g, 7, 4, 64).to(DEV), (1 + 0.1 * randn(g, 64)).to(DEV)
    up = [randn(g, 7, 4, 64).to(DEV) for _ in range(2)]
    table = table_of(64, 7).to(DEV)
    x1, x2, w1, w2 = (t.clone().requires_grad_() for t in (x, x, w, w))
    x, w = x.requires_grad_(), w.requires_grad_()
    a, b = torch.autograd.grad(rotary.kernel_fn(x1, x2, table), (x1, x2), up)
    assert torch.equal(torch.autograd.grad(rotary.kernel_fn(x, x, table), x, up)[0], a + b)
    a, b, c, d = torch.autograd.grad(qk_norm_rotary.kernel_fn(x1, x2, w1, w2, table), (x1, x2, w1, w2), up)
    dx, dw = torch.autograd.grad(qk_norm_rotary.kernel_fn(x, x, w, w, table), (x, w), up)
    assert torch.equal(dx, a + b) and torch.equal(dw, c + d)
    pages, lens, starts, total = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in make_batch([7], [7], 8, 1))
    cache = torch.zeros(total, 8, 4, 64, device=DEV)
    with pytest.raises(ValueError, match="same place"):
        paged_append.kernel_fn(x.detach(), x.detach(), cache, cache, pages, lens, starts)
    # the halves of one allocation are two caches; lengths and starts out of a wider table
    both = torch.zeros(total, 2, 8, 4, 64, device=DEV)
    wide = torch.stack([lens, lens + 1], 1)[:, 0], torch.stack([starts, starts], 1)[:, 0]
    paged_append.kernel_fn(x.detach(), up[0], both[:, 0], both[:, 1], pages, *wide)
    assert torch.equal(both[int(pages[0, 0]), 0, :7], x.detach()) and torch.equal(both[int(pages[0, 0]), 1, :7], up[0])


def test_captured_backward():
    """Forward and backward in one graph, replayed over new values with eager work between."""
    need_gpu()
    from kernels.hip import qk_norm_rotary, rotary
    g = torch.Generator().manual_seed(12)
    dtype = torch.bfloat16
    q, k = randn(g, 70, 4, 64).to(dtype).to(DEV), randn(g, 70, 2, 64).to(dtype).to(DEV)
    wq, wk = ((1 + 0.1 * randn(g, 64)).to(dtype).to(DEV) for _ in range(2))
    gq, gk = randn(g, 70, 4, 64).to(dtype).to(DEV), randn(g, 70, 2, 64).to(dtype).to(DEV)
    table = table_of(64, 70).to(DEV)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]

    def step():
        a, b = qk_norm_rotary.kernel_fn(*leaves, table)
        c, d = rotary.kernel_fn(a, b, table)
        return [c, d, *torch.autograd.grad((c, d), leaves, (gq, gk))]

    say("warm")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        say("replay", i)
        with torch.no_grad():
            q.copy_(randn(g, 70, 4, 64))
            gk.copy_(randn(g, 70, 2, 64))
        want = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_host_forms():
    """The native host side and the Python one give the same bits, with the same autograd contract."""
    need_gpu()
    from kernels.hip import _lib, paged_append, paged_attention, qk_norm_rotary, rotary
    g = torch.Generator().manual_seed(16)
    dtype = torch.bfloat16
    q, k = randn(g, 2, 9, 4, 64).to(dtype).to(DEV), randn(g, 2, 9, 2, 64).to(dtype).to(DEV)
    wq, wk = (1 + 0.1 * randn(g, 64)).to(dtype).to(DEV), (1 + 0.1 * randn(g, 64)).to(dtype).to(DEV)
    table, pos = table_of(32, 40).to(DEV), torch.randint(0, 40, (2, 9), generator=g).to(DEV)
    pages, lens, starts, total = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in make_batch([12, 6], [20, 6], 8, 17))
    caches = [torch.zeros(total, 8, 2, 64, dtype=dtype, device=DEV) for _ in range(2)]
    ups = [randn(g, 2, 9, 4, 64).to(dtype).to(DEV), randn(g, 2, 9, 2, 64).to(dtype).to(DEV)]

    def run():
        out = []
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        for p in (pos, None):
            y = rotary.kernel_fn(*leaves[:2], table, p, interleaved=True)
            out += [*y, *torch.autograd.grad(y, leaves[:2], ups)]
            y = qk_norm_rotary.kernel_fn(*leaves, table, p)
            out += [*y, *torch.autograd.grad(y, leaves, ups)]
        y, none = qk_norm_rotary.kernel_fn(leaves[0], None, leaves[2], None)
        assert none is None
        out += [y, *torch.autograd.grad(y, (leaves[0], leaves[2]), ups[0])]
        y = rotary.kernel_fn(leaves[0], None, table)[0]
        # (an expanded gradient, and a transposed one)
        out += [*torch.autograd.grad(y.sum(), leaves[0], retain_graph=True),
                *torch.autograd.grad((y.transpose(1, 3) * ups[0].transpose(1, 3).contiguous()).sum(), leaves[0])]
        flat_q, flat_k = q.view(18, 4, 64), k.view(18, 2, 64)
        with torch.no_grad():
            r = paged_append.kernel_fn(flat_k, flat_k, *caches, pages, lens, starts, q=flat_q, q_weight=wq, k_weight=wk, table=table)
        out += [r, *(c.clone() for c in caches)]
        out.append(paged_attention.kernel_fn(r, *caches, pages, lens, starts, window=7, softcap=9.0))
        assert not any(t.requires_grad for t in out[-4:])
        return out

    say("native")
    native = run()
    real = _lib.native
    try:
        _lib.native = lambda *t: None
        say("python")
        python = run()
    finally:
        _lib.native = real
    assert len(native) == len(python)
    assert all(torch.equal(a, b) and a.requires_grad == b.requires_grad for a, b in zip(native, python))
    x = q.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(qk_norm_rotary.kernel_fn(x, None, wq, None)[0].float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention.kernel_fn(x.view(18, 4, 64), *caches, pages, lens, starts)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_append.kernel_fn(k.view(18, 2, 64).requires_grad_(), k.view(18, 2, 64), *caches, pages, lens, starts)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(q.detach(), torch.ones_like(q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotary.kernel_fn(d, None, table)
    with torch.inference_mode():
        flat_k = k.view(18, 2, 64).clone()
        paged_append.kernel_fn(flat_k, flat_k, *(c.clone() for c in caches), pages, lens, starts)
    version = caches[0]._version
    paged_append.kernel_fn(k.detach().view(18, 2, 64), k.detach().view(18, 2, 64), *caches, pages, lens, starts)
    assert caches[0]._version > version


def training_calls():
    from kernels.hip import qk_norm_rotary, rotary
    g = torch.Generator().manual_seed(21)
    dtype = torch.bfloat16
    q, k = randn(g, 2, 9, 4, 64).to(dtype).to(DEV), randn(g, 2, 9, 2, 64).to(dtype).to(DEV)
    wq, wk = ((1 + 0.1 * randn(g, 64)).to(dtype).to(DEV) for _ in range(2))
    table, at = table_of(32, 40).to(DEV), torch.randint(0, 40, (2, 9), generator=g).to(DEV)
    return {
        "rotary": ((q, k), lambda q, k: rotary.kernel_fn(q, k, table, at)),
        "rotary one": ((q,), lambda q: rotary.kernel_fn(q, None, table)[:1]),
        "norm": ((q, k, wq, wk), lambda q, k, wq, wk: qk_norm_rotary.kernel_fn(q, k, wq, wk, table, at)),
        "norm one": ((q, wq), lambda q, wq: qk_norm_rotary.kernel_fn(q, None, wq, None)[:1]),
    }


CALLS = ["rotary", "rotary one", "norm", "norm one"]


@pytest.mark.parametrize("name", CALLS)
def test_under_torch_compile(name):
    need_gpu()
    import torch._dynamo
    import torch._dynamo.compiled_autograd as compiled
    leaves, fn = training_calls()[name]
    say("compile", name)
    leaves = [a.requires_grad_() for a in leaves]
    loss = lambda outs: sum((o.float() * o.detach().float()).sum() for o in outs)  # noqa: E731
    outs = fn(*leaves)
    want = [*outs, *torch.autograd.grad(loss(outs), leaves)]
    torch._dynamo.reset()
    outs = torch.compile(fn, backend="eager")(*leaves)
    got = [*outs, *torch.autograd.grad(loss(outs), leaves)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    total = loss(fn(*leaves))
    with compiled._enable(torch.compile(backend="eager")):
        total.backward()
    torch._dynamo.reset()
    for a, b in zip(leaves, want[len(outs):]):
        assert torch.equal(a.grad, b)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    need_gpu()
    import torch.autograd.forward_ad as fw
    leaves, fn = training_calls()[name]
    say("forward mode", name)
    for i in range(len(leaves)):
        for grad_mode in (True, False):
            with fw.dual_level(), torch.set_grad_enabled(grad_mode):
                args = list(leaves)
                args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*args)


@pytest.mark.parametrize("name", ["rotary", "norm"])
def test_parts_of_the_gradient(name):
    """A loss of one output, a gradient of one leaf, tensors saved on the host, two backward passes."""
    need_gpu()
    leaves, fn = training_calls()[name]
    say("parts", name)
    leaves = [a.requires_grad_() for a in leaves]
    up = [torch.randn_like(a) for a in leaves[:2]]
    outs = fn(*leaves)
    both = torch.autograd.grad(outs, leaves, up, retain_graph=True)
    for i in (0, 1):
        alone = torch.autograd.grad(outs[i], leaves, up[i], retain_graph=True, allow_unused=True)
        for j, (a, b) in enumerate(zip(alone, both)):
            if j % 2 == i:
                assert torch.equal(a, b)
            else:
                assert a is None or not a.any()
    for i, leaf in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(outs, leaf, up, retain_graph=True)[0], both[i])
        rest = [a.detach() if a is not leaf else a for a in leaves]
        o = fn(*rest)
        used = [(x, u) for x, u in zip(o, up) if x.requires_grad]
        assert torch.equal(torch.autograd.grad([x for x, _ in used], leaf, [u for _, u in used])[0], both[i])
    with torch.autograd.graph.save_on_cpu():
        o = fn(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, up), both))


def test_serving_under_torch_compile():
    need_gpu()
    import torch._dynamo
    from kernels.hip import paged_append, paged_attention
    say("compile", "serving")
    g = torch.Generator().manual_seed(22)
    x = randn(g, 18, 8, 64).to(torch.bfloat16).to(DEV)
    table = table_of(64, 40).to(DEV)
    pages, lens, starts, total = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in make_batch([12, 6], [20, 6], 8, 17))

    def step(x, kc, vc):
        q = paged_append.kernel_fn(x[:, 4:6], x[:, 6:], kc, vc, pages, lens, starts, q=x[:, :4], table=table)
        return paged_attention.kernel_fn(q, kc, vc, pages, lens, starts)

    made = []
    for fn in (step, torch.compile(step, backend="eager")):
        caches = [torch.zeros(total, 8, 2, 64, dtype=x.dtype, device=DEV) for _ in range(2)]
        made.append([fn(x, *caches), *caches])
    torch._dynamo.reset()
    assert all(torch.equal(a, b) for a, b in zip(*made))
