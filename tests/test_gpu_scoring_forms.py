"""The scoring operators' two host forms on the GPU: the native one and the
Python one give the same bits, under hooks, on other streams, captured, and
where one of them declines."""

import pytest
import torch

from gpu_util import gpu, need_gpu, say

pytestmark = gpu
DEV = "cuda"


def ops(dtype):
    """Three calls, each from leaves to a list of outputs that have gradients (and the rest)."""
    from kernels.hip import lmhead_logprobs, token_logprobs, topk_distillation
    g = torch.Generator().manual_seed(1)
    x = (3 * torch.randn(2, 5, 3001, generator=g)).to(dtype).to(DEV)
    t = torch.randint(0, 3001, (2, 5), generator=g).to(DEV)
    t[0, 1] = -100
    tv, ti = torch.randn(2, 5, 20, generator=g).to(DEV), torch.randint(0, 3001, (2, 5, 20), generator=g).to(DEV)
    half = dtype if dtype != torch.float32 else torch.bfloat16
    h = torch.randn(2, 5, 128, generator=g).to(half).to(DEV)
    w = (0.1 * torch.randn(3001, 128, generator=g)).to(half).to(DEV)

    def logprobs(x):
        r = token_logprobs.kernel_fn(x, t, temperature=0.7, top_k=9)
        return [r.logprobs, r.entropy], [r.top_logprobs, r.top_ids]

    def entropy(x):
        return [token_logprobs.kernel_fn(x, softcap=20.0).entropy], []

    def distill(x):
        return [topk_distillation.kernel_fn(x, tv, ti, temperature=2.0)], []

    def distill_rows(x):
        return [topk_distillation.kernel_fn(x, tv, ti, reduction="none")], []

    def head(h, w):
        return list(lmhead_logprobs.kernel_fn(h, w, t, softcap=30.0)), []

    return [(logprobs, [x]), (entropy, [x]), (distill, [x]), (distill_rows, [x]), (head, [h, w])]


def both(fn, leaves):
    leaves = [a.detach().clone().requires_grad_() for a in leaves]
    outs, rest = fn(*leaves)
    ups = [torch.randn(o.shape, generator=torch.Generator().manual_seed(4)).to(DEV) for o in outs]
    return [*outs, *rest, *torch.autograd.grad(outs, leaves, ups)], (outs, leaves, ups)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_native_and_python_forms_agree(dtype, monkeypatch):
    need_gpu()
    from kernels.hip import _lib
    for fn, leaves in ops(dtype):
        say("forms", dtype, fn.__name__)
        native, _ = both(fn, leaves)
        with torch.no_grad():
            outs, rest = fn(*leaves)
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(outs + rest, native))
        with monkeypatch.context() as m:
            m.setattr(_lib, "native", lambda *a: None)
            python, _ = both(fn, leaves)
        assert len(native) == len(python)
        for a, b in zip(native, python):
            assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b), fn.__name__


def test_native_backward_is_once_differentiable_and_repeats():
    need_gpu()
    for fn, leaves in ops(torch.bfloat16):
        say("repeat", fn.__name__)
        first, (outs, ls, ups) = both(fn, leaves)
        outs, _ = fn(*ls)
        a = torch.autograd.grad(outs, ls, ups, retain_graph=True)
        b = torch.autograd.grad(outs, ls, ups, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(outs, ls, ups, create_graph=True)


def test_saved_tensor_hooks_and_changed_inputs():
    need_gpu()
    for fn, leaves in ops(torch.float16):
        say("hooks", fn.__name__)
        want, _ = both(fn, leaves)
        # hooks that hand back another layout of every matrix
        pack = lambda t: t.cpu()
        unpack = lambda t: t.to(DEV).t().contiguous().t() if t.dim() == 2 else t.to(DEV)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got, _ = both(fn, leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # a saved input changed in place is noticed
        ls = [a.detach().clone().requires_grad_() for a in leaves]
        outs, _ = fn(*ls)
        with torch.no_grad():
            ls[0].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(outs[0].sum(), ls)


def test_side_stream_and_capture():
    """A forward and backward on a side stream, and captured in a graph that is
    replayed with eager work between the replays."""
    need_gpu()
    for fn, leaves in ops(torch.bfloat16):
        say("stream", fn.__name__)
        want, _ = both(fn, leaves)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got, _ = both(fn, leaves)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got
        torch.cuda.synchronize()
        ls = [a.detach().clone().requires_grad_() for a in leaves]
        ups = [torch.randn(o.shape, generator=torch.Generator().manual_seed(4)).to(DEV) for o in fn(*ls)[0]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs, rest = fn(*ls)
            grads = torch.autograd.grad(outs, ls, ups)
        kept = [*(o.detach() for o in outs), *rest, *grads]
        for i in range(3):
            for o in kept:
                o.fill_(3)
            torch.cuda.synchronize()
            say("replay", fn.__name__, i)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, want))
            again, _ = both(fn, leaves)
            assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_declined_calls_and_errors():
    need_gpu()
    from kernels.hip.lmhead_logprobs import kernel_fn as head
    from kernels.hip.token_logprobs import kernel_fn as logprobs
    from kernels.hip.topk_distillation import kernel_fn as distill
    x = torch.randn(6, 100, device=DEV)
    t = torch.randint(0, 100, (6,), device=DEV)
    want = logprobs(x, t)
    for other in (x.t().contiguous().t(), torch.cat([x, x], 1)[:, :100]):
        assert torch.equal(logprobs(other, t.int()).logprobs, want.logprobs)
    assert torch.equal(logprobs(x[:1].expand(6, 100), t).entropy, logprobs(x[:1].repeat(6, 1), t).entropy)
    y = x[:1].clone().requires_grad_()  # a broadcast input: its gradient is the sum over the rows
    (gy,) = torch.autograd.grad(logprobs(y.expand(6, 100), t).logprobs.sum(), y)
    z = x[:1].repeat(6, 1).requires_grad_()
    (gz,) = torch.autograd.grad(logprobs(z, t).logprobs.sum(), z)
    assert torch.equal(gy, gz.sum(0, keepdim=True))
    with pytest.raises(RuntimeError, match="devices|GPU"):
        logprobs(x, t.cpu())
    with pytest.raises(ValueError, match="tokens"):
        logprobs(x, t[:5])
    with pytest.raises(ValueError, match="top_k"):
        logprobs(x, t, top_k=101)
    with pytest.raises(ValueError, match="temperature"):
        logprobs(x, t, temperature=0)
    with pytest.raises(ValueError, match="teacher_ids"):
        distill(x, x[:, :4].contiguous(), t[:, None].expand(6, 3).contiguous())
    with pytest.raises(ValueError, match="go with"):
        head(x, x[:, :64].contiguous(), t)
    with pytest.raises(ValueError, match="chunk_size"):
        head(x.half(), x.half(), t, chunk_size=0)
