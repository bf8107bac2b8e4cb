"""Attention over the paged cache on the GPU, against float64."""

import math

import pytest
import torch

from gpu_util import gpu, need_gpu, say
from heads_util import attend_bound, close, make_batch
from oracle import heads as oracle

pytestmark = gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# counts, lengths, page, q heads, kv heads, dim, window, softcap
CASES = [
    ([1], [1], 16, 1, 1, 64, 0, 0.0),
    ([1], [777], 16, 4, 4, 64, 0, 0.0),
    ([1, 1, 1, 1], [1, 64, 65, 300], 16, 8, 2, 128, 0, 0.0),
    ([1, 1], [513, 2], 48, 6, 2, 80, 0, 30.0),
    ([7], [7], 8, 4, 1, 64, 0, 0.0),
    ([40, 1, 0, 13], [40, 200, 50, 77], 16, 6, 2, 128, 0, 0.0),
    ([150], [150], 16, 2, 2, 64, 0, 0.0),
    ([90, 70], [300, 70], 32, 8, 2, 128, 50, 0.0),
    ([33, 2], [129, 66], 1, 3, 1, 256, 7, 20.0),
    ([130], [161], 7, 5, 1, 72, 0, 0.0),
    ([5, 3], [3, 40], 16, 2, 1, 64, 0, 0.0),          # a sequence shorter than its new tokens
    ([2, 1], [0, 5], 16, 2, 1, 64, 0, 0.0),           # an empty one
    ([3], [50], 16, 32, 1, 96, 1, 0.0),               # many heads share one; each token sees itself alone
    ([70, 70], [70, 100], 64, 12, 4, 192, 64, 0.0),
    ([9, 1], [20, 31], 16, 2, 1, 66, 0, 0.0),         # heads off the vectors
    ([4], [19], 5, 2, 2, 320, 0, 0.0),                # wide heads
    ([1] * 130, [1 + (37 * i) % 90 for i in range(130)], 16, 4, 2, 64, 0, 0.0),
    ([1] * 1500, [(7 * i) % 45 for i in range(1500)], 16, 2, 1, 64, 0, 0.0),   # more sequences than one workgroup lines up
    ([1, 2], [70, 31], 16, 40, 1, 64, 0, 0.0),        # groups past one tile's 32 rows,
    ([2, 1], [45, 9], 16, 130, 1, 256, 0, 0.0),       # past the tiles of wide heads,
    ([1, 2], [45, 9], 16, 300, 1, 64, 0, 0.0),        # past every tile
    ([1, 70], [3003, 2001], 16, 4, 2, 256, 0, 0.0),   # long rows, cut among workers: many of them,
    ([1, 3, 2], [2500, 900, 1], 16, 8, 2, 192, 0, 30.0),   # few of them,
    ([7], [9001], 64, 2, 1, 128, 0, 0.0),             # one tile in very many parts
    ([98], [5000], 128, 1, 1, 256, 0, 0.0),
    ([1, 70], [1503, 901], 16, 4, 2, 64, 333, 20.0),  # a window over many units, cut among workers
    ([5, 1], [90, 33], 16, 2, 1, 128, 0, 0.001),      # caps from the smallest
    ([5, 1], [90, 33], 16, 2, 1, 128, 0, 256.0),
    ([5, 1], [90, 33], 16, 2, 1, 128, 0, 300.0),
    ([5, 1], [90, 33], 16, 2, 1, 66, 0, 10000.0),     # to the largest
    ([4500], [4500], 16, 1, 1, 64, 40, 0.0),          # (with the hint 1: more tiles than sequences explain)
]


def setup(case, dtype, seed=1, sharp=2.0, tail=2):
    counts, lengths, page, hq, hk, dim, window, softcap = case
    g = torch.Generator().manual_seed(seed)
    pages, lens, starts, total = make_batch(counts, lengths, page, seed)
    q = (sharp * torch.randn(sum(counts) + tail, hq, dim, generator=g)).to(dtype)
    kc = torch.randn(total, page, hk, dim, generator=g).to(dtype)
    vc = torch.randn(total, page, hk, dim, generator=g).to(dtype)
    return q, kc, vc, pages, lens, starts


def hide(kc, vc, pages, lens, value):
    """Put `value` into every place that no sequence has."""
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for p in range(n):
            used[int(pages[b, p // kc.shape[1]]), p % kc.shape[1]] = True
    kc[~used] = value
    vc[~used] = value


def check(case, dtype, got, q, kc, vc, pages, lens, starts, scale=None):
    counts, lengths, page, hq, hk, dim, window, softcap = case
    scale = 1 / math.sqrt(dim) if scale is None else scale
    want, spread, reach, mass = oracle.attend(q, kc, vc, pages, lens, starts, scale, softcap, window, bounds=True)
    close(got, want, attend_bound(want, spread, reach, mass, max(lengths + [1]), dim, dtype, softcap), str(case))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c[2:]) + "-" + str(sum(c[0])))
def test_attention(case, dtype):
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    say("attention", case, dtype)
    q, kc, vc, pages, lens, starts = setup(case, dtype)
    hide(kc, vc, pages, lens, math.nan)
    counts, _, _, _, _, _, window, softcap = case
    args = [t.to(DEV) for t in (q, kc, vc, pages, lens, starts)]
    got = kernel_fn(*args, window=window, softcap=softcap)
    assert got.shape == q.shape and got.dtype == dtype and not got[sum(counts):].any()
    check(case, dtype, got, q, kc, vc, pages, lens, starts)
    # hints change the kernel, not the result's rules; out keeps the rows of no sequence
    for hint in (1, max(counts)):
        out = torch.full_like(args[0], 3.0)
        assert kernel_fn(*args, window=window, softcap=softcap, max_chunk=hint, out=out) is out
        assert (out[sum(counts):] == 3).all()
        check(case, dtype, torch.cat([out[:sum(counts)], got[sum(counts):]]), q, kc, vc, pages, lens, starts)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides(dtype):
    """[pages, heads, page, dim] caches, queries inside a fused projection, a strided output."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    case = ([3, 60], [90, 61], 16, 4, 2, 64, 0, 0.0)
    say("strides", dtype)
    q, kc, vc, pages, lens, starts = setup(case, dtype, tail=0)
    fused = torch.zeros(63, 8, 64, dtype=dtype, device=DEV)
    fused[:, 2:6] = q.to(DEV)
    wide = torch.zeros(63, 8, 64, dtype=dtype, device=DEV)
    kt, vt = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (kc, vc))
    p = torch.full((2, 40), 7, dtype=torch.int32, device=DEV)
    p[:, :pages.shape[1]] = pages.to(DEV)
    got = kernel_fn(fused[:, 2:6], kt, vt, p[:, :pages.shape[1]], lens.to(DEV), starts.to(DEV), out=wide[:, 4:])
    check(case, dtype, got, q, kc, vc, pages, lens, starts)
    assert not wide[:, :4].any()
    # one element off the alignment
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)[1:].view(q.shape).copy_(q)
    check(case, dtype, kernel_fn(odd, kt, vt, pages.to(DEV), lens.to(DEV), starts.to(DEV)), q, kc, vc, pages, lens, starts)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("chunk", [1, 100])
def test_long(dtype, chunk):
    """Keys cut over many workers, a page table wider than the sequences."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    case = ([chunk, chunk], [5003, 1201], 16, 4, 1, 128, 0, 0.0)
    say("long", dtype, chunk)
    q, kc, vc, pages, lens, starts = setup(case, dtype, tail=0)
    wide = torch.full((2, 4000), -1, dtype=torch.int32)
    wide[:, :pages.shape[1]] = pages
    got = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, wide, lens)))
    again = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, wide, lens)))
    assert torch.equal(got, again)
    rows = list(range(0, 2 * chunk, 17 if chunk > 1 else 1))
    full = oracle.sequences(lens.tolist(), None, 2 * chunk)
    for t in rows:  # a token alone is a batch of one
        b, p = full[t]
        one = torch.tensor([p + 1], dtype=torch.int32)
        check(([1], [p + 1], 16, 4, 1, 128, 0, 0.0), dtype, got[t:t + 1], q[t:t + 1], kc, vc, wide[b:b + 1], one, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_hidden_values(dtype):
    """Infinities and NaN in keys and values of later tokens, of keys past the window and of
    pages that are not there reach no row that does not see them."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    g = torch.Generator().manual_seed(3)
    for count, n, window in ((40, 40, 0), (40, 150, 30), (1, 150, 30), (3, 100, 0), (200, 200, 0)):
        case = ([count], [n], 16, 4, 2, 64, window, 0.0)
        say("hidden", case, dtype)
        q, kc, vc, pages, lens, starts = setup(case, dtype, tail=0)
        clean = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens, starts)), window=window)
        for value in (math.nan, math.inf, -math.inf):
            k2, v2 = kc.clone(), vc.clone()
            last = n - 1  # seen by the last token alone
            if count > 1:
                k2[int(pages[0, last // 16]), last % 16] = value
                v2[int(pages[0, last // 16]), last % 16] = value
            first = n - count - window if window else None  # the last key that no token sees
            if first is not None and first >= 0:
                k2[int(pages[0, first // 16]), first % 16] = value
                v2[int(pages[0, first // 16]), first % 16] = value
            got = kernel_fn(*(t.to(DEV) for t in (q, k2, v2, pages, lens, starts)), window=window)
            rows = slice(0, count - 1) if count > 1 else slice(0, 1)
            assert torch.equal(got[rows], clean[rows]), (case, value)
            if count > 1:
                assert not torch.isfinite(got[-1]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_scores_at_the_edges(dtype):
    """Scores far apart, equal, infinite; a NaN query; the type's lowest value as a mask."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    case = ([4], [40], 16, 2, 1, 64, 0, 0.0)
    say("edges", dtype)
    q, kc, vc, pages, lens, starts = setup(case, dtype, sharp=30.0, tail=0)
    place = [(int(pages[0, p // 16]), p % 16) for p in range(40)]

    def run(q, kc, vc, **kw):
        return kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens, starts)), **kw)

    check(case, dtype, run(q, kc, vc), q, kc, vc, pages, lens, starts)
    zero = torch.zeros_like(q)
    check(case, dtype, run(zero, kc, vc), zero, kc, vc, pages, lens, starts)  # the mean of the values
    # keys whose scores are -inf leave their places; all of them: 0
    k2 = kc.clone()
    one = torch.ones_like(q)
    for p in range(0, 40, 3):
        k2[place[p]] = -math.inf
    check(case, dtype, run(one, k2, vc), one, k2, vc, pages, lens, starts)
    for p in range(40):
        k2[place[p]] = -math.inf
    assert not run(one, k2, vc).any()
    # +inf or NaN among the seen scores: a NaN row
    k2 = kc.clone()
    k2[place[37]] = math.inf
    got = run(one, k2, vc)
    assert torch.isnan(got[1:]).all() and torch.isfinite(got[0]).all()
    assert torch.isfinite(run(one, k2, vc, softcap=20.0)).all()
    q2 = q.clone()
    q2[2, 1, 5] = math.nan
    got = run(q2, kc, vc)
    assert torch.isnan(got[2, 1]).all() and torch.isfinite(got[2, 0]).all() and torch.isfinite(got[3]).all()
    # products near the type's lowest value: finite scores beside it win alone
    low = torch.finfo(dtype).min
    q3, k3 = torch.zeros_like(q), torch.zeros_like(kc)
    q3[..., 0], k3[..., 0] = 1.0, low
    k3[place[3]][:] = 0.0
    got = run(q3, k3, vc, scale=1.0)
    close(got, vc[place[3]].double().expand(4, 2, 64), torch.zeros(4, 2, 64), "lowest")


@pytest.mark.parametrize("dim", [4, 8])
def test_more_rows_than_a_grid(dim):
    """Past 2^20 rows, of which each sees its own key alone: the values come back as they are."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    counts, page, dtype = [2 ** 20 + 77, 0, 300], 64, torch.bfloat16
    say("many rows", dim)
    pages, lens, starts, total = make_batch(counts, counts, page, 4)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(sum(counts) + 1, 1, dim, generator=g).to(dtype).to(DEV)
    kc, vc = (torch.randn(total, page, 1, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    pages = pages.to(DEV)
    got = kernel_fn(q, kc, vc, pages, lens.to(DEV), starts.to(DEV), window=1)
    place = torch.arange(counts[0], device=DEV)
    assert torch.equal(got[:counts[0]], vc[pages[0, place // page].long(), place % page])
    place = torch.arange(counts[2], device=DEV)
    assert torch.equal(got[counts[0]:-1], vc[pages[2, place // page].long(), place % page])
    assert not got[-1].any()


def test_bad_pages_and_batches():
    """Pages outside the cache hide their keys; lengths past the table's width are cut;
    starts out of range or order stay inside the tensors."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    for dtype in DTYPES:
        case = ([3, 40], [90, 100], 16, 4, 2, 64, 0, 0.0)
        say("bad pages", dtype)
        q, kc, vc, pages, lens, starts = setup(case, dtype, tail=0)
        pages[0, 2], pages[1, 0], pages[1, 3] = -7, kc.shape[0], 2 ** 31 - 1
        got = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens, starts)))
        check(case, dtype, got, q, kc, vc, pages, lens, starts)
        none = torch.full_like(pages, -1)
        assert not kernel_fn(*(t.to(DEV) for t in (q, kc, vc, none, lens, starts))).any()
        say("bad lengths", dtype)
        for values in ([2 ** 31 - 1, 10 ** 6], [-5, -2 ** 31], [0, 0]):
            got = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages)), torch.tensor(values, dtype=torch.int32, device=DEV),
                            starts.to(DEV))
            assert torch.isfinite(got).all() and (got.any() or values[0] <= 0)
        say("bad starts", dtype)
        for values in ([0, 50, 43], [-9, 2 ** 31 - 1, 3], [43, 0, 0], [7, 7, 7], [20, 30, 25]):
            got = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens)), torch.tensor(values, dtype=torch.int32, device=DEV))
            assert torch.isfinite(got).all()
        say("no sequences, no tokens, no pages", dtype)
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
        assert not kernel_fn(q.to(DEV), kc.to(DEV), vc.to(DEV), z(0, 3), z(0), z(1)).any()
        assert kernel_fn(q[:0].to(DEV), kc.to(DEV), vc.to(DEV), z(0, 3), z(0)).shape == (0, 4, 64)
        assert not kernel_fn(q.to(DEV), kc[:0].to(DEV), vc[:0].to(DEV), pages.to(DEV), lens.to(DEV), starts.to(DEV)).any()
        assert not kernel_fn(q.to(DEV), kc.to(DEV), vc.to(DEV), z(2, 0), lens.to(DEV), starts.to(DEV)).any()


def test_shared_pages():
    """Sequences that share the pages of a common beginning read what their own copies would give."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    dtype = torch.bfloat16
    say("shared pages")
    q, kc, vc, pages, lens, starts = setup(([1, 1, 1], [100, 100, 100], 16, 4, 2, 64, 0, 0.0), dtype, tail=0)
    for i in range(4):
        for b in (1, 2):
            kc[int(pages[b, i])], vc[int(pages[b, i])] = kc[int(pages[0, i])], vc[int(pages[0, i])]
    apart = kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens)))
    pages[1:, :4] = pages[0, :4]
    assert torch.equal(kernel_fn(*(t.to(DEV) for t in (q, kc, vc, pages, lens))), apart)


def test_a_far_place_in_a_large_cache():
    """Element offsets past 2^32 (a cache of 9 GB, of which a few pages are touched)."""
    need_gpu()
    from kernels.hip import paged_append, paged_attention
    dtype = torch.bfloat16
    pages = 2 ** 32 // (16 * 2 * 128) + 9
    say("far place")
    kc = torch.empty(pages, 16, 2, 128, dtype=dtype, device=DEV)
    vc = torch.empty(pages, 16, 2, 128, dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(40, 2, 128, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(40, 4, 128, generator=g).to(dtype)
    at = torch.tensor([[pages - 1, 3, pages - 5]], dtype=torch.int32)
    lens = torch.tensor([40], dtype=torch.int32)
    paged_append.kernel_fn(k.to(DEV), v.to(DEV), kc, vc, at.to(DEV), lens.to(DEV))
    for hint in (1, 40):
        got = paged_attention.kernel_fn(q.to(DEV), kc, vc, at.to(DEV), lens.to(DEV), torch.tensor([0, 40], dtype=torch.int32, device=DEV),
                                        max_chunk=hint)
        small_k, small_v = (torch.zeros(3, 16, 2, 128, dtype=dtype) for _ in range(2))
        for p in range(40):
            small_k[p // 16, p % 16], small_v[p // 16, p % 16] = k[p], v[p]
        check(([40], [40], 16, 4, 2, 128, 0, 0.0), dtype, got, q, small_k, small_v, torch.tensor([[0, 1, 2]]), lens, None)


def test_a_step_of_a_model():
    """Prompts, then decode steps, through the cache: norm, rotation, append and attention
    against causal attention over the whole sequences."""
    need_gpu()
    from kernels.hip import paged_append, paged_attention, qk_norm_rotary
    from kernels.hip.rotary import rotary_table
    g = torch.Generator().manual_seed(6)
    dtype, hq, hk, dim, page = torch.bfloat16, 4, 2, 64, 16
    final = [37, 20, 50]
    prompt = [30, 1, 45]
    x = [torch.randn(n, hq + 2 * hk, dim, generator=g).to(dtype) for n in final]
    wq, wk = (1 + 0.1 * torch.randn(dim, generator=g)).to(dtype), (1 + 0.1 * torch.randn(dim, generator=g)).to(dtype)
    table = rotary_table(dim, 64)
    pages, _, _, total = make_batch([1] * 3, final, page, 7)
    pages = pages.to(DEV)
    kc = torch.full((total, page, hk, dim), math.nan, dtype=dtype, device=DEV)
    vc = torch.full_like(kc, math.nan)
    have, outs = [0, 0, 0], [[], [], []]
    steps = [prompt] + [[1, 3, 1]] * 5 + [[2, 4, 0]]
    for counts in steps:
        new = torch.cat([x[b][have[b]:have[b] + c] for b, c in enumerate(counts)]).to(DEV)
        have = [h + c for h, c in zip(have, counts)]
        lens = torch.tensor(have, dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, counts[0], counts[0] + counts[1], sum(counts)], dtype=torch.int32, device=DEV)
        say("step", counts)
        q = paged_append.kernel_fn(new[:, hq:hq + hk], new[:, hq + hk:], kc, vc, pages, lens, starts, q=new[:, :hq],
                                   q_weight=wq.to(DEV), k_weight=wk.to(DEV), table=table.to(DEV))
        o = paged_attention.kernel_fn(q, kc, vc, pages, lens, starts, max_chunk=max(counts))
        for b in range(3):
            outs[b].append(o[int(starts[b]):int(starts[b + 1])])
    assert have == final
    for b, n in enumerate(final):
        # the same heads as training's operator gives, then attention in float64 over them
        q, k = qk_norm_rotary.kernel_fn(x[b][:, :hq].to(DEV), x[b][:, hq:hq + hk].to(DEV), wq.to(DEV), wk.to(DEV), table.to(DEV))
        cut = -(-n // page) * page
        kk, vv = torch.zeros(cut, hk, dim, dtype=dtype), torch.zeros(cut, hk, dim, dtype=dtype)
        kk[:n], vv[:n] = k.cpu(), x[b][:, hq + hk:]
        own = torch.arange(cut // page, dtype=torch.int32)[None]
        check(([n], [n], page, hq, hk, dim, 0, 0.0), dtype, torch.cat(outs[b]), q.cpu(), kk.view(-1, page, hk, dim),
              vv.view(-1, page, hk, dim), own, torch.tensor([n], dtype=torch.int32), None)


def test_streams_and_graphs():
    """On another stream; two captured calls of different batches, replayed in turn with lengths
    that grow and eager calls between."""
    need_gpu()
    from kernels.hip.paged_attention import kernel_fn
    dtype = torch.bfloat16
    made = []
    for counts, lengths in (([1] * 5, [3, 700, 64, 129, 2000]), ([30, 1, 90], [500, 900, 90])):
        q, kc, vc, pages, lens, starts = (t.to(DEV) for t in setup((counts, lengths, 16, 8, 2, 128, 0, 0.0), dtype, tail=1))
        made.append((q, kc, vc, pages, lens, starts))
    say("eager")
    eager = [kernel_fn(*a) for a in made]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [kernel_fn(*a) for a in made]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs, outs = [], []
    for a in made:
        say("capture")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernel_fn(*a))
        graphs.append(graph)
    for i in range(3):
        for a in made:
            a[4].sub_(1)  # shorter by one
        want = [kernel_fn(*a) for a in made]
        for o in outs:
            o.fill_(5.0)
        torch.cuda.synchronize()
        say("replay", i)
        for graph in graphs:
            graph.replay()
        kernel_fn(*made[i % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
